"""A policy over discrete tokens from the framework's operators: embedder, RMSNorm, gated block, head; trained towards a
teacher's top logits and sampled from.  Each stage is checked in float64 against what that stage read on the GPU."""

import math

import pytest
import torch

from robolearn_amd import kernels as K
from robolearn_amd.config import FlashSACConfig
from robolearn_amd.networks import FlatStore, FusedOptimizer
from test_gpu_sample import reference_row

pytestmark = pytest.mark.gpu


class TokenPolicy:
    """logits = (act(n Wg^T) * (n Wu^T)) Wd^T + e, times Wh^T, with e = x We^T and n = RMSNorm(e)."""

    def __init__(self, inputs, width, hidden, classes, rows, entries, device, bf16):
        shapes = {"embed": (width, inputs), "norm": (width,), "gated": (2, hidden, width), "down": (width, hidden),
                  "head": (classes, width)}
        self.store = FlatStore(shapes, device, shadows=bf16)
        g = torch.Generator().manual_seed(width)
        for name, view in self.store.params().items():
            value = torch.ones(shapes[name]) if name == "norm" else torch.randn(shapes[name], generator=g) / math.sqrt(shapes[name][-1])
            view.copy_(value)
        self.store.refresh_shadows()
        self.optimizer = FusedOptimizer(self.store, FlashSACConfig(learning_rate_init=1e-3), plain=True, schedule=False)
        self.p, self.grad = self.store.params(), self.store.grads()
        self.w = self.store.shadows() if bf16 else self.p
        self.mode = K.BF16 if bf16 else K.FP32_SPLIT
        kind = torch.bfloat16 if bf16 else torch.float32
        self.sizes = inputs, width, hidden, classes, rows

        def buf(*shape, dtype=kind):
            return torch.zeros(*shape, dtype=dtype, device=device)

        f32 = torch.float32
        self.x, self.xh = buf(rows, inputs, dtype=f32), buf(rows, inputs)
        self.e, self.n32, self.n = buf(rows, width, dtype=f32), buf(rows, width, dtype=f32), buf(rows, width)
        self.ms, self.partial = buf(rows, dtype=f32), buf(64 * width, dtype=f32)
        self.h, self.y, self.yh = buf(rows, hidden), buf(rows, width, dtype=f32), buf(rows, width)
        self.logits, self.dlogits = buf(rows, classes, dtype=f32), buf(rows, classes, dtype=f32)
        self.dlh, self.dy, self.dyh = buf(rows, classes), buf(rows, width, dtype=f32), buf(rows, width)
        self.dh32, self.dh, self.dn, self.de, self.deh = (buf(rows, hidden, dtype=f32), buf(rows, hidden), buf(rows, width),
                                                          buf(rows, width, dtype=f32), buf(rows, width))
        self.dn32 = buf(rows, width, dtype=f32)
        self.loss = buf(rows, dtype=f32)
        self.ws = buf(max(K.gated_workspace(rows, width, hidden, kind, backward=True), 1 << 22), dtype=torch.uint8)
        self.teacher, self.index = buf(rows, entries, dtype=f32), buf(rows, entries, dtype=torch.int64)
        self.uniform, self.tokens, self.log_probs = (buf(rows, dtype=f32), buf(rows, dtype=torch.int64), buf(rows, dtype=f32))
        self.bf16 = bf16

    def _half(self, source, destination):
        if self.bf16:
            K.cast_bf16(source, destination)
            return destination
        return source

    def forward(self):
        inputs, width, hidden, classes, rows = self.sizes
        linear = dict(rows=rows, mode=self.mode)
        K.linear_forward(self._half(self.x, self.xh), self.w["embed"], self.e, in_dim=inputs, out_dim=width, **linear)
        K.rms_forward(self.e, self.p["norm"], self.ms, self.n32, rows=rows, channels=width)
        K.gated_forward(self._half(self.n32, self.n), self.w["gated"], self.h, activation="silu", workspace=self.ws)
        K.linear_forward(self.h, self.w["down"], self.y, in_dim=hidden, out_dim=width, c=self.e, beta=1.0, **linear)
        K.linear_forward(self._half(self.y, self.yh), self.w["head"], self.logits, in_dim=width, out_dim=classes, **linear)

    def act(self):
        self.forward()
        K.categorical_sample(self.logits, self.uniform, self.tokens, temperature=0.9, top_k=20, top_p=0.95, log_probs=self.log_probs)

    def train(self):
        inputs, width, hidden, classes, rows = self.sizes
        both = dict(rows=rows, mode=self.mode)
        self.forward()
        K.distill_forward(self.logits, self.teacher, self.index, self.loss, temperature=2.0, dlogits=self.dlogits,
                          grad_scale=1.0 / rows)
        dl = self._half(self.dlogits, self.dlh)
        y, n, x = (self.yh, self.n, self.xh) if self.bf16 else (self.y, self.n32, self.x)
        K.linear_backward_weight(dl, y, self.grad["head"], in_dim=width, out_dim=classes, **both)
        K.linear_backward_input(dl, self.w["head"], self.dy, in_dim=width, out_dim=classes, **both)
        dy = self._half(self.dy, self.dyh)
        K.linear_backward_weight(dy, self.h, self.grad["down"], in_dim=hidden, out_dim=width, **both)
        K.linear_backward_input(dy, self.w["down"], self.dh32, in_dim=hidden, out_dim=width, **both)
        dh = self._half(self.dh32, self.dh)
        K.gated_backward(n, self.w["gated"], dh, self.dn, self.grad["gated"], activation="silu", workspace=self.ws)
        self.dn32.copy_(self.dn)
        self.de.copy_(self.dy)
        K.rms_backward(self.e, self.dn32, self.p["norm"], self.ms, self.partial, self.de, self.grad["norm"], rows=rows,
                       channels=width, accumulate_dx=True)
        K.linear_backward_weight(self._half(self.de, self.deh), x, self.grad["embed"], in_dim=inputs, out_dim=width, **both)
        self.optimizer.step()


def fill(policy, seed):
    g = torch.Generator().manual_seed(seed)
    inputs, _, _, classes, rows = policy.sizes
    policy.x.copy_(torch.randn(rows, inputs, generator=g))
    teacher, index = torch.topk(2 * torch.randn(rows, classes, generator=g), policy.teacher.shape[1], 1)
    index[::5, -2:] = -1
    policy.teacher.copy_(teacher)
    policy.index.copy_(index)
    policy.uniform.copy_(torch.rand(rows, generator=g))


def make(gpu, bf16, seed=1, sizes=(39, 96, 264, 301, 150)):
    policy = TokenPolicy(*sizes, 12, gpu, bf16)
    fill(policy, seed)
    return policy


def close(got, exact, magnitude, k, stored, kind):
    """A sum of k products, each as exact as its operands: (k / 16 + 40) 2^-23 of the products' absolute sum (the
    three-piece products drop as much again), plus `stored` roundings to `kind` on the way."""
    bound = magnitude * ((math.ceil(k / 16) + 40) * 2.0**-23 + stored * torch.finfo(kind).eps / 2) + 1e-30
    assert ((got.double().cpu() - exact).abs() <= bound).all()


@pytest.mark.parametrize("bf16", [False, True])
def test_stages_and_gradients(gpu, bf16):
    policy = make(gpu, bf16)
    before = {k: v.clone() for k, v in policy.p.items()}
    kind = torch.bfloat16 if bf16 else torch.float32
    weights = {k: v.double().cpu() for k, v in policy.w.items()}
    policy.train()
    torch.cuda.synchronize()
    inputs, width, hidden, classes, rows = policy.sizes
    d = lambda t: t.double().cpu()  # noqa: E731
    x, n, y, dl, dy, dh, de = ((policy.xh, policy.n, policy.yh, policy.dlh, policy.dyh, policy.dh, policy.deh) if bf16 else
                               (policy.x, policy.n32, policy.y, policy.dlogits, policy.dy, policy.dh32, policy.de))
    close(policy.e, d(x) @ weights["embed"].t(), d(x).abs() @ weights["embed"].t().abs(), inputs, 0, kind)
    gate, up = d(n) @ weights["gated"][0].t(), d(n) @ weights["gated"][1].t()
    sig = torch.sigmoid(gate)
    value, slope = gate * sig, sig * (1 + gate * (1 - sig))
    size_g, size_u = (d(n).abs() @ weights["gated"][i].t().abs() for i in (0, 1))
    # |silu'| <= 1.1, |silu''| <= 0.5; exp and its quotient 2^-21
    close(policy.h, value * up, 1.1 * size_g * up.abs() + value.abs() * size_u + 4 * (value * up).abs(), width, 1, kind)
    close(policy.y, d(policy.h) @ weights["down"].t() + d(policy.e),
          d(policy.h).abs() @ weights["down"].t().abs() + d(policy.e).abs(), hidden, 0, kind)
    close(policy.logits, d(y) @ weights["head"].t(), d(y).abs() @ weights["head"].t().abs(), width, 0, kind)

    loss, grad = 0.0, torch.zeros(rows, classes, dtype=torch.float64)
    z, index = d(policy.logits) / 2.0, policy.index.cpu()
    for r in range(rows):
        valid = index[r] >= 0
        p = torch.softmax(d(policy.teacher)[r][valid] / 2.0, 0)
        log_q = torch.log_softmax(z[r], 0)
        row_loss = 4.0 * (p * (p.log() - log_q[index[r][valid]])).sum()
        # logarithms of size up to 40, each to 2^-22
        assert abs(policy.loss[r].item() - row_loss) <= 4 * 40 * 2.0**-22
        grad[r] = log_q.exp()
        grad[r].index_add_(0, index[r][valid], -p)
    grad *= 2.0 / rows
    assert ((d(policy.dlogits) - grad).abs() <= 2.0**-17 * (2.0 / rows)).all()

    def product(got, a, b, k, stored=0):
        close(got, a @ b, a.abs() @ b.abs(), k, stored, kind)

    product(policy.grad["head"], d(dl).t(), d(y), rows)
    product(policy.dy, d(dl), weights["head"], classes)
    product(policy.grad["down"], d(dy).t(), d(policy.h), rows)
    product(policy.dh32, d(dy), weights["down"], width)
    dg, du = d(dh) * up * slope, d(dh) * value
    # dg and du come from sums over `width`, and are stored once; |slope| <= 1.1, |slope'| <= 0.5
    slack = (math.ceil(width / 16) + 40) * 2.0**-23
    e_dg = d(dh).abs() * (size_u * 1.1 + up.abs() * (0.5 * size_g + 4)) * slack + dg.abs() * torch.finfo(kind).eps / 2
    e_du = d(dh).abs() * (1.1 * size_g + 4 * value.abs()) * slack + du.abs() * torch.finfo(kind).eps / 2
    for got, a, e, b, k in ((policy.dn, torch.cat((dg, du), 1), torch.cat((e_dg, e_du), 1), weights["gated"].flatten(0, 1), 2 * hidden),
                            (policy.grad["gated"], torch.cat((dg, du), 1).t(), torch.cat((e_dg, e_du), 1).t(), d(n), rows)):
        exact = a @ b
        bound = (e @ b.abs() + (math.ceil(k / 16) + 40) * 2.0**-23 * ((a.abs() + e) @ b.abs())) * 1.01 + \
            exact.abs() * torch.finfo(got.dtype).eps / 2 * 1.01 + 1e-30
        assert ((d(got).reshape(exact.shape) - exact).abs() <= bound).all()
    product(policy.grad["embed"], d(de).t(), d(x), rows)
    # Adam's first step is the learning rate against the gradient's sign, where the gradient outweighs eps
    for name, view in policy.p.items():
        step, g = (view - before[name]).cpu(), policy.grad[name].cpu()
        big = g.abs() > 1e-4
        assert big.any() and (step[big] / -g[big].sign() - 1e-3).abs().max() <= 1e-3 * 1e-3 + 2.0**-22


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("sizes", [(39, 96, 264, 301, 150), (8, 64, 128, 2500, 1)])
def test_acting(gpu, bf16, sizes):
    policy = make(gpu, bf16, sizes=sizes)
    policy.act()
    logits, u = policy.logits.cpu().numpy(), policy.uniform.cpu()
    for r in range(sizes[-1]):
        token, log_prob = reference_row(logits[r], u[r].item(), temperature=0.9, top_k=20, top_p=0.95)
        assert policy.tokens[r] == token and abs(policy.log_probs[r].item() - log_prob) <= 2.0**-24 * abs(log_prob) + 1e-12


def test_training_and_acting_in_one_graph(gpu):
    """The captured step, replayed with eager work between the replays, gives what eager steps give."""
    eager, captured = make(gpu, True), make(gpu, True)
    captured.train()  # kernels are loaded before the capture
    captured.act()
    captured = make(gpu, True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured.train()
        captured.act()
    for seed in (3, 4, 5):
        for policy in (eager, captured):
            fill(policy, seed)
        eager.train()
        eager.act()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(eager.store.param, captured.store.param) and torch.equal(eager.loss, captured.loss)
        assert torch.equal(eager.tokens, captured.tokens) and torch.equal(eager.log_probs, captured.log_probs)
        assert torch.equal(eager.store.grad, captured.store.grad)


def test_offsets_past_32_bits(gpu):
    """Rows that begin past the 2^31st element of their tensor."""
    rows, classes = 70000, 32768
    z = torch.zeros(rows, classes, dtype=torch.bfloat16, device=gpu)
    z[-2:] = 3 * torch.randn(2, classes, generator=torch.Generator().manual_seed(1)).bfloat16().to(gpu)
    tokens, u = torch.empty(rows, dtype=torch.int64, device=gpu), torch.full((rows,), 0.37, device=gpu)
    K.categorical_sample(z, u, tokens, top_p=0.9)
    for r in (rows - 2, rows - 1):
        assert tokens[r] == reference_row(z[r].float().cpu().numpy(), u[r].item(), top_p=0.9)[0]
    teacher, index = torch.zeros(rows, 4, device=gpu), torch.arange(4, device=gpu).repeat(rows, 1)
    loss, alone, few = torch.empty(rows, device=gpu), torch.empty(2, device=gpu), z[-2:].clone()
    expected = torch.empty_like(few)
    K.distill_forward(few, teacher[:2].contiguous(), index[:2].contiguous(), alone, dlogits=expected)
    K.distill_forward(z, teacher, index, loss, dlogits=z)
    assert torch.equal(loss[-2:], alone) and torch.equal(z[-2:], expected)
    del z
    # a row pitch of 2^20 values
    rows, inputs, hidden, pitch = 2100, 72, 40, 1 << 20
    g = torch.Generator().manual_seed(2)
    x = torch.randn(rows, inputs, generator=g).bfloat16().to(gpu)
    w = torch.randn(2, hidden, inputs, generator=g).bfloat16().to(gpu)
    dh = torch.randn(rows, hidden, generator=g).bfloat16().to(gpu)
    store = torch.empty(rows * pitch, dtype=torch.bfloat16, device=gpu)
    outputs = []
    for step in (inputs, pitch, pitch + 1 if (rows - 1) * (pitch + 1) + inputs <= rows * pitch else pitch):
        far = store.as_strided((rows, inputs), (step, 1))
        far.copy_(x)
        h, dx, dw = torch.empty(rows, hidden, dtype=torch.bfloat16, device=gpu), torch.empty_like(x), torch.empty_like(w)
        ws = torch.empty(K.gated_workspace(rows, inputs, hidden, torch.bfloat16, backward=True), dtype=torch.uint8, device=gpu)
        K.gated_forward(far, w, h, workspace=ws)
        K.gated_backward(far, w, dh, dx, dw, workspace=ws)
        outputs.append((h, dx, dw))
    for other in outputs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(outputs[0], other))


@pytest.mark.parametrize("operator", ["gated", "distill", "sample"])
def test_another_stream(gpu, operator):
    """Calls on a stream of the caller's, after work that it waits for, on tensors of the default stream."""
    g = torch.Generator().manual_seed(4)
    z = torch.randn(64, 5000, generator=g).to(gpu)
    stream = torch.cuda.Stream()
    results = []
    for side in (False, True):
        source = torch.zeros_like(z)
        out = torch.empty_like(z)
        rows = torch.empty(64, device=gpu)
        tokens = torch.empty(64, dtype=torch.int64, device=gpu)
        w = torch.ones(2, 24, 5000, device=gpu) / 70
        h = torch.empty(64, 24, device=gpu)
        ws = torch.empty(K.gated_workspace(64, 5000, 24, torch.float32), dtype=torch.uint8, device=gpu)
        teacher, index = torch.zeros(64, 3, device=gpu), torch.arange(3, device=gpu).repeat(64, 1)
        u = torch.full((64,), 0.7, device=gpu)
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream if side else torch.cuda.current_stream()):
            source.copy_(z)
            if operator == "gated":
                K.gated_forward(source, w, h, workspace=ws)
            elif operator == "distill":
                K.distill_forward(source, teacher, index, rows, dlogits=out)
            else:
                K.categorical_sample(source, u, tokens)
        torch.cuda.synchronize()
        results.append({"gated": [h], "distill": [rows, out], "sample": [tokens]}[operator])
    assert all(torch.equal(a, b) for a, b in zip(*results))
