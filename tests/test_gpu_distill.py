"""Distillation from a teacher's top logits against float64."""

import math

import pytest
import torch

from robolearn_amd import kernels as K

pytestmark = pytest.mark.gpu

# (rows, classes, entries): one class, action bins, odd vocabularies, either side of each kernel's row length
SHAPES = [(1, 1, 1), (3, 2, 2), (9, 101, 16), (5, 255, 64), (6, 257, 1), (7, 513, 300), (5, 1000, 64), (4, 2049, 1024),
          (3, 4099, 33), (3, 20011, 50), (2, 33000, 64), (2, 65537, 20), (2, 131072, 64), (2, 140001, 5)]
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def reference(z, t, index, weights, temperature):
    """Loss, logsumexp and the gradient of the losses' sum, row by row in float64."""
    rows, classes = z.shape
    loss, grad, lse = torch.zeros(rows, dtype=torch.float64), torch.zeros(rows, classes, dtype=torch.float64), []
    for r in range(rows):
        log_q = torch.log_softmax(z[r].double() / temperature, 0)
        lse.append(torch.logsumexp(z[r].double() / temperature, 0))
        valid = (index[r] >= 0) & (index[r] < classes)
        if weights[r] == 0 or not valid.any():
            continue
        log_p = torch.log_softmax(t[r][valid].double() / temperature, 0)
        p, at = log_p.exp(), index[r][valid].long()
        loss[r] = weights[r] * temperature**2 * torch.where(p > 0, p * (log_p - log_q[at]), 0).sum()
        grad[r] = log_q.exp()
        grad[r].index_add_(0, at, -p)
        grad[r] *= weights[r] * temperature
    return loss, torch.stack(lse), grad


def inputs(rows, classes, entries, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    z = (3 * torch.randn(rows, classes, generator=g)).to(dtype)
    t = 2 * torch.randn(rows, entries, generator=g)
    index = torch.stack([torch.randperm(max(classes, entries), generator=g)[:entries] for _ in range(rows)])  # some outside
    index[torch.rand(rows, entries, generator=g) < 0.2] = -1
    weights = torch.rand(rows, generator=g)
    if rows > 2:
        weights[1] = 0
        index[2] = -1  # a row without entries
    if entries > 1:
        index[0, 1] = index[0, 0]  # a class named twice
    return z, t, index, weights


def bounds(z, t, index, loss, lse, grad, weights, temperature, dtype):
    """An exponent (x - max) / T is off by 3 2^-24 of itself and exp2 by 2^-23; a sum of n values in a fixed order of
    threads by (n / 64 + 32) 2^-24.  Every q and p is off by that, relatively; the loss by p times the logarithms' own
    size; lse by 2^-24 of itself; then one rounding to the output's type."""
    classes, entries = z.shape[1], t.shape[1]
    x = z.double() / temperature
    span = (x.amax(1, keepdim=True) - x).clamp(max=100) + x.abs().clamp(max=100) * 2.0**-10
    log_q = x - lse[:, None]
    rel_q = (3 * span + classes / 64 + 64) * 2.0**-24
    rel_p = (3 * ((t.amax(1) - t.amin(1)) / temperature) + entries / 64 + 64) * 2.0**-24
    weight = (weights.double() * temperature)[:, None]
    q = log_q.exp() * (weight != 0)
    d = weight * (q * rel_q) + (weight * q - grad).abs() * rel_p.double()[:, None]
    half = torch.finfo(dtype).eps / 2
    tiny = 2.0**-25 if dtype == torch.float16 else 1e-37
    grad_bound = d + half * (grad.abs() + d) + 2.0**-23 * (weight * q + grad.abs()) + tiny
    size = 1 + log_q.abs().amax(1) + (t.amax(1) - t.amin(1)).double() / temperature + math.log(entries)
    loss_bound = weights.double() * temperature**2 * size * (rel_p.double() + rel_q.amin(1) + 2.0**-20)
    return loss_bound + 1e-30, grad_bound


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pad,temperature,wide", [(0, 1.0, True), (3, 2.5, False)])
@pytest.mark.parametrize("rows,classes,entries", SHAPES)
def test_distill_against_float64(gpu, rows, classes, entries, pad, temperature, wide, dtype):
    print(f"case distill {rows}x{classes} entries={entries} pad={pad} {dtype}", flush=True)
    z, t, index, weights = inputs(rows, classes, entries, dtype, classes + entries)
    if not wide:
        index = index.int()
    loss, lse, grad = reference(z, t, index, weights, temperature)
    store = torch.full((rows + 1, classes + pad), float("nan"), dtype=dtype)
    store[:rows, :classes] = z
    store = store.to(gpu)
    zd = store[:rows, :classes]
    td, indexd, weightsd = t.to(gpu), index.to(gpu), weights.to(gpu)
    out = torch.full((rows + 1, classes + pad), 7.0, dtype=dtype, device=gpu)
    dz = out[:rows, :classes]
    rows_out, lse_out = torch.empty(rows, device=gpu), torch.empty(rows, device=gpu)
    K.distill_forward(zd, td, indexd, rows_out, temperature=temperature, weights=weightsd, lse=lse_out, dlogits=dz)
    torch.cuda.synchronize()
    loss_bound, grad_bound = bounds(z, t, index, loss, lse, grad, weights, temperature, dtype)
    assert ((rows_out.cpu().double() - loss).abs() <= loss_bound).all()
    assert ((lse_out.cpu().double() - lse).abs() <= 2.0**-23 * lse.abs() + (classes / 64 + 64) * 2.0**-24).all()
    assert ((dz.cpu().double() - grad).abs() <= grad_bound).all()
    assert (out[rows:] == 7).all() and (out[:, classes:] == 7).all()

    # the loss alone, and the gradient from row gradients; lse's rounding moves every q by 2^-24 |lse|
    again = torch.empty(rows, device=gpu)
    K.distill_forward(zd, td, indexd, again, temperature=temperature, weights=weightsd)
    assert torch.equal(again, rows_out)
    dloss = torch.linspace(-1.5, 1.5, rows)
    out.fill_(7.0)
    K.distill_backward(zd, td, indexd, lse_out, dloss.to(gpu), dz, temperature=temperature, weights=weightsd)
    scale = dloss.double()[:, None]
    q = (z.double() / temperature - lse[:, None]).exp() * (weights.double() * temperature)[:, None]
    extra = q * ((2 * lse.abs() + 4 * (z.double() / temperature).abs().clamp(max=100).amax(1))[:, None] * 2.0**-23)
    assert ((dz.cpu().double() - scale * grad).abs() <= scale.abs() * (grad_bound + extra) + (1e-37 if dtype != torch.float16 else 2.0**-25)).all()
    assert (out[rows:] == 7).all() and (out[:, classes:] == 7).all()

    # in the logits' place
    expected = torch.empty(rows, classes, dtype=dtype, device=gpu)
    K.distill_forward(zd, td, indexd, rows_out, temperature=temperature, weights=weightsd, dlogits=expected, grad_scale=0.5)
    K.distill_forward(zd, td, indexd, rows_out, temperature=temperature, weights=weightsd, dlogits=zd, grad_scale=0.5)
    assert torch.equal(zd, expected) and torch.equal(again, rows_out)
    assert store[rows:].isnan().all() and store[:, classes:].isnan().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("classes", [101, 5000, 70000])
def test_masked_and_invalid_values(gpu, classes, dtype):
    """Masked classes (-inf) outside the teacher's entries have no gradient; inside them the loss is infinite.  Rows of
    weight 0, or without a teacher, may hold anything.  A NaN in a row that counts makes that row NaN alone."""
    g = torch.Generator().manual_seed(classes)
    rows, entries = 8, 4
    z = torch.randn(rows, classes, generator=g).to(dtype)
    t = torch.randn(rows, entries, generator=g)
    index = torch.arange(entries).repeat(rows, 1) * 7
    weights = torch.ones(rows)
    z[0, 50:] = -math.inf
    z[1, 7] = -math.inf
    z[2] = math.nan
    weights[2] = 0
    t[3, 1] = -math.inf
    z[3, 7] = -math.inf            # the entry's probability is 0: no term
    z[4, 90] = math.nan
    t[5] = -math.inf               # a teacher that says nothing
    z[5, 3] = math.nan
    t[6, 2] = math.nan
    loss, grad = torch.full((rows,), 7.0, device=gpu), torch.full((rows, classes), 7.0, dtype=dtype, device=gpu)
    K.distill_forward(z.to(gpu), t.to(gpu), index.to(gpu), loss, weights=weights.to(gpu), dlogits=grad)
    loss, grad = loss.cpu(), grad.cpu()
    assert math.isfinite(loss[0]) and (grad[0, 50:] == 0).all() and grad[0].isfinite().all()
    assert loss[1] == math.inf and grad[1].isfinite().all() and grad[1, 7] < 0
    assert loss[2] == 0 and (grad[2] == 0).all()
    expected, _, exact = reference(z[3:4], t[3:4], index[3:4], weights[3:4], 1.0)
    assert abs(loss[3].double() - expected[0]) <= 2.0**-16 and grad[3].isfinite().all() and grad[3, 7] == 0
    assert loss[4].isnan() and loss[6].isnan()
    assert loss[5] == 0 and (grad[5] == 0).all()
    expected, _, _ = reference(z[7:], t[7:], index[7:], weights[7:], 1.0)
    assert abs(loss[7].double() - expected[0]) <= 2.0**-16


def test_distill_gradient_against_differences(gpu):
    """fp32, step 2^-5 along a direction: the third-order term is bounded by the float64 function's own, the rounding of
    the two losses by 2^-20 of their logarithms' size over the step."""
    rows, classes, entries, temperature = 6, 300, 20, 1.7
    z, t, index, weights = inputs(rows, classes, entries, torch.float32, 11)
    v = torch.randn(rows, classes, generator=torch.Generator().manual_seed(1))
    step = 2.0**-5

    def loss(s):
        out = torch.empty(rows, device=gpu)
        K.distill_forward((z + s * v).to(gpu), t.to(gpu), index.to(gpu), out, temperature=temperature, weights=weights.to(gpu))
        return out.cpu().double()

    def loss64(s):
        return reference(z.double() + s * v.double(), t, index, weights, temperature)[0]

    out, grad = torch.empty(rows, device=gpu), torch.empty(rows, classes, device=gpu)
    K.distill_forward(z.to(gpu), t.to(gpu), index.to(gpu), out, temperature=temperature, weights=weights.to(gpu), dlogits=grad)
    slope = (grad.cpu().double() * v.double()).sum(1)
    third = ((loss64(2 * step) - 2 * loss64(step) + 2 * loss64(-step) - loss64(-2 * step)) / (2 * step**3)).abs()
    bound = 2 * third * step**2 / 6 + temperature**2 * 40 * 2.0**-20 / step
    assert ((loss(step) - loss(-step)) / (2 * step) - slope).abs().le(bound).all()


@pytest.mark.parametrize("rows,classes", [(0, 40), (37, 101), (5, 40000)])
def test_distill_in_a_graph(gpu, rows, classes):
    z, t, index, weights = (v.to(gpu) for v in inputs(max(rows, 1), classes, 8, torch.bfloat16, 4))
    z, t, index, weights = z[:rows], t[:rows], index[:rows], weights[:rows]
    other = z.flip(0).contiguous()
    loss, grad = torch.empty(rows, device=gpu), torch.empty_like(z)

    def step():
        K.distill_forward(z, t, index, loss, weights=weights, dlogits=grad)

    results = []
    kept = z.clone()
    for source in (kept, other):
        z.copy_(source)
        step()
        results.append((loss.clone(), grad.clone()))
    if rows == 0:
        return
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in (0, 1, 0):
        z.copy_((kept, other)[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(loss, results[i][0]) and torch.equal(grad, results[i][1])
