"""Gated feed-forward products and their gradients against float64."""

import math

import pytest
import torch

from robolearn_amd import kernels as K

pytestmark = pytest.mark.gpu

# (rows, inputs, hidden): one token, edges of the tiles and of the 64-deep steps, odd widths, more than one tile
SHAPES = [(1, 1, 1), (1, 64, 64), (1, 1032, 520), (2, 8, 3), (5, 39, 17), (16, 128, 200), (17, 72, 264), (63, 64, 65),
          (64, 123, 100), (130, 160, 129), (257, 65, 136), (300, 200, 256)]
TYPES = [torch.bfloat16, torch.float16, torch.float32]


BEHIND = 1 << 16  # bytes behind a buffer that a test looks at


def workspace_for(x, w, gpu, backward):
    need = K.gated_workspace(x.shape[0], x.shape[1], w.shape[1], x.dtype, backward=backward)
    return torch.full((need + BEHIND,), 0xff, dtype=torch.uint8, device=gpu)[:need]  # NaN in every type


def flat(shape, dtype, gpu):
    """A contiguous tensor of sevens, and what lies behind it."""
    values = math.prod(shape)
    store = torch.full((values + BEHIND,), 7.0, dtype=dtype, device=gpu)
    return store[values:], store[:values].view(shape)


def behind(workspace):
    return workspace.as_strided((BEHIND,), (1,), workspace.storage_offset() + workspace.numel())


def activation64(g, act):
    if act == "relu":
        return g.clamp(min=0), (g > 0).double()
    if act == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    phi = torch.special.ndtr(g)
    return g * phi, phi + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)


def padded(values, pad, gpu):
    """values [rows, columns] on the GPU in rows of columns + pad, NaN in the pad and in a row behind the last."""
    rows, columns = values.shape
    store = torch.full((rows + 1, columns + pad), float("nan"), dtype=values.dtype)
    store[:rows, :columns] = values
    return store.to(gpu)[:rows, :columns]


def guarded(rows, columns, pad, dtype, gpu):
    store = torch.full((rows + 1, columns + pad), 7.0, dtype=dtype, device=gpu)
    return store, store[:rows, :columns]


def untouched(store, rows, columns):
    return (store[rows:] == 7).all() and (store[:, columns:] == 7).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act,pad", [("silu", 0), ("gelu", 3), ("relu", 8)])
@pytest.mark.parametrize("rows,inputs,hidden", SHAPES)
def test_gated_against_float64(gpu, rows, inputs, hidden, act, pad, dtype):
    """Bounds: a projection of K values adds at most K / 16 + 4 times 2^-23 of its row's times its column's norm (matrix
    accumulations of 16; the three-piece products of fp32 drop 2^-23 more); exp and the activation add (|g| + 8) 2^-22
    relative; every value that is stored in the operands' type is rounded by eps / 2 (subnormal fp16: 2^-25).  dg and
    du are stored so, then summed against |w| or |x|."""
    print(f"case gated {rows}x{inputs}x{hidden} {act} pad={pad} {dtype}", flush=True)
    g = torch.Generator().manual_seed(rows + 7 * inputs + 31 * hidden)
    x = torch.randn(rows, inputs, generator=g).to(dtype)
    w = (torch.randn(2, hidden, inputs, generator=g) / math.sqrt(inputs)).to(dtype)
    dh = torch.randn(rows, hidden, generator=g).to(dtype)
    xd, dhd, wd = padded(x, pad, gpu), padded(dh, pad, gpu), w.to(gpu)
    h_store, h = guarded(rows, hidden, pad, dtype, gpu)
    dx_store, dx = guarded(rows, inputs, pad, dtype, gpu)
    past_dw, dw = flat((2, hidden, inputs), dtype, gpu)
    spaces = [workspace_for(x, w, gpu, backward) for backward in (False, True)]
    K.gated_forward(xd, wd, h, activation=act, workspace=spaces[0])
    K.gated_backward(xd, wd, dhd, dx, dw, activation=act, workspace=spaces[1])
    torch.cuda.synchronize()
    assert (past_dw == 7).all() and all((behind(space) == 0xff).all() for space in spaces)

    x64, w64, dh64 = x.double(), w.double(), dh.double()
    gate, up = x64 @ w64[0].t(), x64 @ w64[1].t()
    value, slope = activation64(gate, act)
    half = torch.finfo(dtype).eps / 2
    tiny = 2.0**-25 if dtype == torch.float16 else 1e-37
    # fp32: the stored value is the fp32 result itself
    sums = math.ceil(inputs / 16) + 8
    norm = x64.norm(dim=1, keepdim=True)
    d_gate, d_up = sums * 2.0**-23 * norm * w64[0].norm(dim=1), sums * 2.0**-23 * norm * w64[1].norm(dim=1)
    rough = (gate.abs() + 8) * 2.0**-22
    # |act'| <= 1.13, |act''| <= 1 (relu: the slope flips where the gate is within its error of 0)
    d_value = 1.13 * d_gate + rough * value.abs()
    d_slope = 1.0 * d_gate + rough
    if act == "relu":
        d_slope = (gate.abs() <= d_gate).double()
    error = d_value * up.abs() + value.abs() * d_up + d_value * d_up
    bound = error + half * ((value * up).abs() + error) + tiny
    assert untouched(h_store, rows, hidden)
    assert ((h.cpu().double() - value * up).abs() <= bound).all()

    dg, du = dh64 * up * slope, dh64 * value
    e_dg = dh64.abs() * (d_up * slope.abs() + up.abs() * d_slope + d_up * d_slope)
    e_du = dh64.abs() * d_value
    e_dg = e_dg + (half + 2.0**-22) * (dg.abs() + e_dg) + tiny
    e_du = e_du + (half + 2.0**-22) * (du.abs() + e_du) + tiny

    def product_bound(a, e_a, b, exact):
        """sum a b with a off by e_a, in fp32 sums of a.shape[1] values, rounded once."""
        magnitude = (a.abs() + e_a) @ b.abs()
        error = e_a @ b.abs() + (math.ceil(a.shape[1] / 16) + 40) * 2.0**-23 * magnitude
        return error + half * (exact.abs() + error) + tiny

    exact = dg @ w64[0] + du @ w64[1]
    bound = product_bound(torch.cat((dg, du), 1), torch.cat((e_dg, e_du), 1), torch.cat((w64[0], w64[1])), exact)
    assert untouched(dx_store, rows, inputs)
    assert ((dx.cpu().double() - exact).abs() <= bound).all()
    for half_w, d, e in ((0, dg, e_dg), (1, du, e_du)):
        exact = d.t() @ x64
        assert ((dw[half_w].cpu().double() - exact).abs() <= product_bound(d.t(), e.t(), x64, exact)).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("inputs,act,pad", [(100, "gelu", 0), (150, "silu", 3), (520, "relu", 8), (1000, "silu", 0)])
def test_two_tiles_a_workgroup(gpu, inputs, act, pad, dtype):
    """512 tiles of 256 x 256 on 256 CUs, ragged at both ends, over 2, 3, 9 and 16 K tiles."""
    test_gated_against_float64(gpu, 8155, inputs, 2043, act, pad, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,inputs,hidden", [(1, 40, 24), (3, 7, 5), (100, 72, 130), (1000, 136, 264), (700, 123, 300),
                                                (2100, 64, 40), (16, 512, 520), (123, 1620, 76), (65, 1001, 1)])
def test_small_integers_are_exact(gpu, rows, inputs, hidden, dtype):
    """Sparse values of -1, 0 and 1 with relu: every sum is a whole number that fp32 holds, dg and du at most 128, so
    the outputs are float64's rounded once.  A missing, doubled or misplaced term shows."""
    print(f"case integers {rows}x{inputs}x{hidden} {dtype}", flush=True)
    g = torch.Generator().manual_seed(rows * inputs + hidden)

    def sparse(*shape, keep):
        v = torch.randint(-1, 2, shape, generator=g) * (torch.rand(shape, generator=g) < keep)
        return v.double()

    keep = min(1.0, 3.0 / math.sqrt(inputs))
    x, w, dh = sparse(rows, inputs, keep=keep), sparse(2, hidden, inputs, keep=keep), sparse(rows, hidden, keep=0.7)
    gate, up = x @ w[0].t(), x @ w[1].t()
    dg, du = dh * up * (gate > 0), dh * gate.clamp(min=0)
    assert max(dg.abs().max(), du.abs().max(), (gate.clamp(min=0) * up).abs().max()) <= 256
    xd, wd, dhd = (t.to(dtype).to(gpu) for t in (x, w, dh))
    h = torch.empty(rows, hidden, dtype=dtype, device=gpu)
    K.gated_forward(xd, wd, h, activation="relu", workspace=workspace_for(xd, wd, gpu, False))
    assert torch.equal(h.cpu().double(), gate.clamp(min=0) * up)
    for dw_type in (dtype, torch.float32):
        dx = torch.empty(rows, inputs, dtype=dtype, device=gpu)
        past_dw, dw = flat((2, hidden, inputs), dw_type, gpu)
        K.gated_backward(xd, wd, dhd, dx, dw, activation="relu", workspace=workspace_for(xd, wd, gpu, True))
        assert (past_dw == 7).all()
        assert torch.equal(dx.cpu(), (dg @ w[0] + du @ w[1]).to(dtype))
        assert torch.equal(dw.cpu(), torch.stack((dg.t() @ x, du.t() @ x)).to(dw_type))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_one_output_alone_and_no_rows(gpu, dtype):
    g = torch.Generator().manual_seed(3)
    x, dh = torch.randn(70, 48, generator=g).to(dtype).to(gpu), torch.randn(70, 90, generator=g).to(dtype).to(gpu)
    w = torch.randn(2, 90, 48, generator=g).to(dtype).to(gpu)
    ws = workspace_for(x, w, gpu, True)
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    K.gated_backward(x, w, dh, dx, dw, workspace=ws)
    dx1, dw1 = torch.empty_like(x), torch.empty_like(w)
    K.gated_backward(x, w, dh, dx1, None, workspace=ws)
    K.gated_backward(x, w, dh, None, dw1, workspace=ws)
    assert torch.equal(dx, dx1) and torch.equal(dw, dw1)
    none = torch.empty(0, 48, dtype=dtype, device=gpu)
    empty = torch.empty(0, 90, dtype=dtype, device=gpu)
    assert K.gated_workspace(0, 48, 90, dtype, backward=True) == 0
    K.gated_forward(none, w, empty)
    K.gated_backward(none, w, empty, none, dw1)
    assert (dw1 == 0).all()


def test_gated_gradient_against_differences(gpu):
    """Central differences of the forward pass in fp32: with a step of 2^-6 the third-order term is at most 2^-12 / 6 of
    the third derivative along the direction, the rounding of the sums 2^-23 sum |h dh| / 2^-6."""
    g = torch.Generator().manual_seed(5)
    rows, inputs, hidden = 40, 24, 56
    x, w = torch.randn(rows, inputs, generator=g), torch.randn(2, hidden, inputs, generator=g) / math.sqrt(inputs)
    dh = torch.randn(rows, hidden, generator=g).to(gpu)
    vx, vw = torch.randn(rows, inputs, generator=g) / 8, torch.randn(2, hidden, inputs, generator=g) / 8
    ws = workspace_for(x, w, gpu, True)

    def loss(step):
        h = torch.empty(rows, hidden, device=gpu)
        K.gated_forward((x + step * vx).to(gpu), (w + step * vw).to(gpu), h, activation="silu", workspace=ws)
        return (h.double() * dh.double()).sum().item(), (h.double() * dh.double()).abs().sum().item()

    step = 2.0**-6
    (plus, size), (minus, _) = loss(step), loss(-step)
    dx, dw = torch.empty(rows, inputs, device=gpu), torch.empty(2, hidden, inputs, device=gpu)
    K.gated_backward(x.to(gpu), w.to(gpu), dh, dx, dw, activation="silu", workspace=ws)
    slope = (dx.cpu().double() * vx).sum().item() + (dw.cpu().double() * vw).sum().item()
    # the same differences of the float64 function bound the third-order term
    def loss64(s):
        a, b = (x + s * vx).double(), (w + s * vw).double()
        gate = a @ b[0].t()
        return (gate * torch.sigmoid(gate) * (a @ b[1].t()) * dh.cpu().double()).sum().item()

    third = abs((loss64(2 * step) - 2 * loss64(step) + 2 * loss64(-step) - loss64(-2 * step)) / (2 * step**3))
    bound = 2 * third * step**2 / 6 + 16 * 2.0**-23 * size / step + 64 * 2.0**-23 * size
    assert abs((plus - minus) / (2 * step) - slope) <= bound


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gated_calls_in_a_graph_and_on_two_streams(gpu, dtype):
    g = torch.Generator().manual_seed(9)
    rows, inputs, hidden = 200, 123, 300
    w = (torch.randn(2, hidden, inputs, generator=g) / 11).to(dtype).to(gpu)
    batches = [(torch.randn(rows, inputs, generator=g).to(dtype).to(gpu), torch.randn(rows, hidden, generator=g).to(dtype).to(gpu))
               for _ in range(3)]

    def buffers(x):
        return (torch.empty(rows, hidden, dtype=dtype, device=gpu), torch.empty_like(x), torch.empty_like(w),
                workspace_for(x, w, gpu, True))

    def step(x, dh, h, dx, dw, ws):
        K.gated_forward(x, w, h, workspace=ws)
        K.gated_backward(x, w, dh, dx, dw, workspace=ws)

    expected = []
    for x, dh in batches:
        out = buffers(x)
        step(x, dh, *out)
        expected.append([t.clone() for t in out[:3]])
    x, dh = (t.clone() for t in batches[0])
    out = buffers(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(x, dh, *out)
    for i in (1, 2, 0):
        x.copy_(batches[i][0])
        dh.copy_(batches[i][1])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out[:3], expected[i]))
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [buffers(x) for _ in range(2)]
    torch.cuda.synchronize()
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            step(*batches[i + 1], *outs[i])
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for a, b in zip(outs[i][:3], expected[i + 1]))
