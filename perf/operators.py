"""Operators of a policy over discrete tokens: the gated feed-forward product, the distillation loss, the sampler.

The cases below measure each operator over the sizes it meets: acting on one environment and on thousands,
minibatches of the training recipes, vocabularies from the bins of one action dimension to 131072 tokens.
``prepare`` makes the inputs and the buffers a program holds, ``run`` makes one pass (the framework's call where
``own`` is true, elementary torch operations otherwise), ``exact`` repeats it in 64 bits.
"""

import math

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one environment's observation through a wide policy's hidden layer: the weights are read once
        dict(name="gated_single", kind="gated", rows=1, inputs=1024, hidden=4096, act="silu", dtype="bf16"),
        # acting on 64 environments with the medium network
        dict(name="gated_envs", kind="gated", rows=64, inputs=512, hidden=2048, act="gelu", dtype="fp16"),
        # the humanoid critic's widths on a full batch, forward and backward
        dict(name="gated_batch", kind="gated", rows=8192, inputs=1024, hidden=4096, act="silu", dtype="bf16"),
        dict(name="gated_batch_backward", kind="gated_backward", rows=8192, inputs=1024, hidden=4096, act="silu",
             dtype="bf16"),
        # an embedder's odd input width (123 observations) on a ragged minibatch
        dict(name="gated_ragged_backward", kind="gated_backward", rows=3001, inputs=123, hidden=1000, act="gelu",
             dtype="fp16"),
        # an fp32 learner's minibatch
        dict(name="gated_fp32_backward", kind="gated_backward", rows=2048, inputs=256, hidden=1024, act="silu",
             dtype="fp32"),
        # a student of action bins on the medium recipe's batch: all latency
        dict(name="distill_bins", kind="distill", rows=2048, classes=101, top=16, dtype="fp32", temperature=1.0),
        # a student with a token vocabulary on a training batch: loss and gradient in one call
        dict(name="distill_tokens", kind="distill", rows=4096, classes=32768, top=64, dtype="bf16", temperature=2.0),
        # the gradient alone from given row gradients, odd vocabulary
        dict(name="distill_odd_backward", kind="distill_backward", rows=1000, classes=50021, top=50, dtype="fp32",
             temperature=1.5),
        # eight action dimensions of 4096 environments, 256 bins each
        dict(name="sample_bins", kind="sample", rows=32768, classes=256, dtype="bf16", top_k=0, top_p=1.0, min_p=0.0,
             by_row=False),
        # one request's next token: all latency
        dict(name="sample_single", kind="sample", rows=1, classes=32768, dtype="fp32", top_k=50, top_p=0.95, min_p=0.0,
             by_row=False),
        # a serving batch whose requests bring their own settings
        dict(name="sample_requests", kind="sample", rows=256, classes=131072, dtype="bf16", top_k=64, top_p=0.9,
             min_p=0.02, by_row=True),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["gated", "gated_backward", "distill", "distill_backward", "sample", "sample"])
    dtype = rng.choice(["bf16", "fp16", "fp32"])
    if kind.startswith("gated"):
        # widths of 8 values a row mostly, as layers have them, and any others
        step = rng.choice([1, 8, 8, 64])
        inputs = max(step, _log_int(rng, 24, 2048) // step * step)
        hidden = max(step, _log_int(rng, 64, 8192) // step * step)
        budget = 8192 * 1024 * 4096 // (16 if dtype == "fp32" else 1)
        rows = _log_int(rng, 1, max(2, min(16384, budget // (inputs * hidden))))
        # in fp32 the slope of relu at a gate next to 0 goes by the order of a sum
        act = rng.choice(["silu", "gelu"] if dtype == "fp32" else ["silu", "gelu", "relu"])
        return dict(kind=kind, rows=rows, inputs=inputs, hidden=hidden, act=act, dtype=dtype)
    if kind.startswith("distill"):
        classes = _log_int(rng, 21, 131072)
        budget = 4096 * 32768 * 2 // (4 if dtype == "fp32" else 2)
        rows = _log_int(rng, 1, max(2, min(32768, budget // classes)))
        return dict(kind=kind, rows=rows, classes=classes, top=min(classes, _log_int(rng, 1, 256)), dtype=dtype,
                    temperature=round(rng.uniform(0.5, 4.0), 3))
    classes = _log_int(rng, 21, 131072)
    budget = 256 * 131072 * 2 // (4 if dtype == "fp32" else 2)
    rows = _log_int(rng, 1, max(2, min(32768, budget // classes)))
    return dict(kind=kind, rows=rows, classes=classes, dtype=dtype, top_k=rng.choice([0, 0, 1, _log_int(rng, 2, 1024)]),
                top_p=rng.choice([1.0, round(rng.uniform(0.3, 0.99), 3)]),
                min_p=rng.choice([0.0, 0.0, round(rng.uniform(0.001, 0.2), 4)]), by_row=rng.random() < 0.5)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEVICE)

    if case["kind"].startswith("gated"):
        rows, inputs, hidden = case["rows"], case["inputs"], case["hidden"]
        state = dict(case=case, x=normal(rows, inputs).to(dtype),
                     w=(normal(2, hidden, inputs) / math.sqrt(inputs)).to(dtype))
        if case["kind"] == "gated":
            state["h"] = torch.empty(rows, hidden, device=DEVICE, dtype=dtype)
        else:
            state["dh"] = normal(rows, hidden).to(dtype)
            state["dx"] = torch.empty(rows, inputs, device=DEVICE, dtype=dtype)
            state["dw"] = torch.empty(2, hidden, inputs, device=DEVICE, dtype=dtype)
        return state

    rows, classes = case["rows"], case["classes"]
    z = 2.0 * normal(rows, classes)
    if case["kind"] == "sample":
        # a policy that knows something: some tokens of each row stand out
        liked = torch.randint(0, classes, (rows, min(32, classes)), generator=g, device=DEVICE)
        z.scatter_add_(1, liked, 4.0 + 2.0 * normal(*liked.shape))
        state = dict(case=case, logits=z.to(dtype), uniform=torch.rand(rows, generator=g, device=DEVICE),
                     tokens=torch.empty(rows, dtype=torch.int64, device=DEVICE),
                     log_probs=torch.empty(rows, device=DEVICE))
        settings = dict(temperature=0.8, top_k=case["top_k"], top_p=case["top_p"], min_p=case["min_p"])
        if case["by_row"]:
            # half of the requests leave a filter off
            def some(value, none, dt=torch.float32):
                on = torch.rand(rows, generator=g, device=DEVICE) < 0.5
                return torch.where(on, torch.full((rows,), value, device=DEVICE, dtype=dt),
                                   torch.full((rows,), none, device=DEVICE, dtype=dt))
            settings = dict(temperature=0.5 + torch.rand(rows, generator=g, device=DEVICE),
                            top_k=some(case["top_k"], 0, torch.int32), top_p=some(case["top_p"], 1.0),
                            min_p=some(case["min_p"], 0.0))
        state["settings"] = settings
        return state

    top = case["top"]
    teacher, index = torch.topk(0.6 * z + 1.5 * normal(rows, classes), top, dim=1)
    # a teacher that stored fewer entries for some rows, and padding rows of weight 0
    kept = torch.randint(max(1, top // 2), top + 1, (rows, 1), generator=g, device=DEVICE)
    index = torch.where(torch.arange(top, device=DEVICE) < kept, index, -1)
    weights = (torch.rand(rows, generator=g, device=DEVICE) < 0.9).float()
    if rows == 1:
        weights.fill_(1.0)
    state = dict(case=case, logits=z.to(dtype), teacher=teacher.contiguous(), index=index, weights=weights,
                 loss=torch.empty(rows, device=DEVICE), dlogits=torch.empty(rows, classes, device=DEVICE, dtype=dtype))
    if case["kind"] == "distill_backward":
        # what the forward pass left behind, and the gradient that reaches each row's loss
        state["lse"] = torch.logsumexp(state["logits"].double() / case["temperature"], 1).float()
        state["dloss"] = normal(rows)
    return state


def run(state):
    return (_own if own else _plain)(state)


def _own(state):
    from robolearn_amd import kernels as K

    case = state["case"]
    kind = case["kind"]
    if kind.startswith("gated"):
        if "workspace" not in state:
            need = K.gated_workspace(case["rows"], case["inputs"], case["hidden"], state["x"].dtype,
                                     backward=kind == "gated_backward")
            state["workspace"] = torch.empty(max(need, 1), dtype=torch.uint8, device=DEVICE)
        if kind == "gated":
            K.gated_forward(state["x"], state["w"], state["h"], activation=case["act"], workspace=state["workspace"])
            return state["h"]
        K.gated_backward(state["x"], state["w"], state["dh"], state["dx"], state["dw"], activation=case["act"],
                         workspace=state["workspace"])
        return state["dx"], state["dw"]
    if kind == "sample":
        K.categorical_sample(state["logits"], state["uniform"], state["tokens"], log_probs=state["log_probs"],
                             **state["settings"])
        return state["tokens"], state["log_probs"]
    if kind == "distill":
        K.distill_forward(state["logits"], state["teacher"], state["index"], state["loss"],
                          temperature=case["temperature"], weights=state["weights"], dlogits=state["dlogits"],
                          grad_scale=1.0)
        return state["loss"], state["dlogits"]
    K.distill_backward(state["logits"], state["teacher"], state["index"], state["lse"], state["dloss"],
                       state["dlogits"], temperature=case["temperature"], weights=state["weights"])
    return state["dlogits"]


def _activation(g, act):
    """act(g) and act'(g)."""
    if act == "relu":
        return torch.clamp(g, min=0), (g > 0).to(g.dtype)
    if act == "silu":
        s = 1 / (1 + torch.exp(-g))
        return g * s, s * (1 + g * (1 - s))
    phi = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
    return g * phi, phi + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))


def _plain(state):
    case = state["case"]
    kind = case["kind"]
    if kind.startswith("gated"):
        x, w = state["x"].float(), state["w"].float()
        gate, up = x @ w[0].t(), x @ w[1].t()
        value, slope = _activation(gate, case["act"])
        if kind == "gated":
            return (value * up).to(state["x"].dtype)
        dh = state["dh"].float()
        dgate, dup = dh * up * slope, dh * value
        dx = dgate @ w[0] + dup @ w[1]
        dw = torch.stack((dgate.t() @ x, dup.t() @ x))
        return dx.to(state["x"].dtype), dw.to(state["x"].dtype)
    if kind == "sample":
        return _plain_sample(state["logits"], state["uniform"], **state["settings"])
    return _plain_distill(state)


def _plain_sample(logits, uniform, temperature, top_k, top_p, min_p):
    """Sums and borders in 64 bits: a token is chosen by comparing long cumulative sums."""
    rows, classes = logits.shape

    def column(v, dtype):
        return (v if torch.is_tensor(v) else torch.full((rows,), v, device=logits.device)).to(dtype)[:, None]

    t, p, least = column(temperature, torch.float64), column(top_p, torch.float64), column(min_p, torch.float64)
    k = column(top_k, torch.int64)
    k = torch.where((k <= 0) | (k > classes), classes, k)
    z, order = torch.sort(logits.float(), dim=1, descending=True, stable=True)
    z = z.double() / t
    weight = torch.exp(z - z[:, :1])
    rank = torch.arange(classes, device=logits.device)
    weight = torch.where(rank < k, weight, 0.0)
    before = torch.cumsum(weight, 1) - weight
    nucleus = (before < p * weight.sum(1, keepdim=True)) | (p >= 1) | (rank == 0)
    weight = torch.where(nucleus & ((weight >= least) | (rank == 0)), weight, 0.0)
    total = weight.sum(1, keepdim=True)
    weight = torch.zeros_like(weight).scatter_(1, order, weight)
    reached = torch.cumsum(weight, 1)
    token = (reached <= uniform.double()[:, None] * total).sum(1).clamp(max=classes - 1)
    chosen = torch.gather(weight, 1, token[:, None])
    return token, torch.log(chosen / total)[:, 0].float()


def _plain_distill(state):
    case = state["case"]
    t = case["temperature"]
    z, index = state["logits"].float() / t, state["index"]
    valid = index >= 0
    entry = torch.where(valid, state["teacher"] / t, -math.inf)
    entry = entry - entry.amax(1, keepdim=True)
    p = torch.exp(entry)
    total = p.sum(1, keepdim=True)
    p = p / total
    safe = index.clamp(min=0)
    if case["kind"] == "distill":
        top = z.amax(1, keepdim=True)
        lse = top + torch.log(torch.exp(z - top).sum(1, keepdim=True))
    else:
        lse = state["lse"][:, None]
    q = torch.exp(z - lse)
    grad = t * (q - torch.zeros_like(q).scatter_add_(1, safe, p))
    scale = state["weights"] if case["kind"] == "distill" else state["weights"] * state["dloss"]
    grad = (grad * scale[:, None]).to(state["logits"].dtype)
    if case["kind"] == "distill_backward":
        return grad
    log_q = torch.gather(z, 1, safe) - lse
    term = torch.where(valid, p * (entry - torch.log(total) - log_q), 0.0)
    return state["weights"] * (t * t) * term.sum(1), grad


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"].startswith("gated"):
        r, i, h = case["rows"], case["inputs"], case["hidden"]
        if case["kind"] == "gated":
            return {"bytes": size * (r * i + 2 * h * i + r * h), "flops": 4 * r * i * h}
        # the two projections again (no activations are handed over), then both gradients
        return {"bytes": size * (2 * r * i + 4 * h * i + r * h), "flops": 12 * r * i * h}
    n = case["rows"] * case["classes"]
    if case["kind"] == "sample":
        settings = 16 if case["by_row"] else 0
        return {"bytes": n * size + case["rows"] * (16 + settings), "flops": 4 * n}
    entries = case["rows"] * case["top"] * 12
    return {"bytes": 2 * n * size + entries + 12 * case["rows"], "flops": 6 * n}


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind.startswith("gated"):
        x, w = state["x"].double(), state["w"].double()
        g, u = torch.matmul(x, w[0].T), torch.matmul(x, w[1].T)
        act = case["act"]
        if act == "silu":
            sig = torch.sigmoid(g)
            a, da = g * sig, sig + g * sig * (1 - sig)
        elif act == "gelu":
            cdf = torch.special.ndtr(g)
            a, da = g * cdf, cdf + g * torch.exp(-g.square() / 2) / math.sqrt(2 * math.pi)
        else:
            a, da = g.relu(), torch.where(g > 0, 1.0, 0.0).double()
        if kind == "gated":
            return a * u
        dh = state["dh"].double()
        pre = torch.cat((dh * u * da, dh * a), dim=1)
        hidden, inputs = case["hidden"], case["inputs"]
        return pre @ w.reshape(2 * hidden, inputs), (pre.T @ x).reshape(2, hidden, inputs)
    if kind == "sample":
        return _exact_sample(state)
    z = state["logits"].double() / case["temperature"]
    rows, classes = z.shape
    valid = state["index"] >= 0
    log_p = torch.log_softmax((state["teacher"].double() / case["temperature"]).masked_fill(~valid, -math.inf), dim=1)
    p = log_p.exp()
    weights = state["weights"].double()
    if kind == "distill":
        log_q = torch.log_softmax(z, dim=1)
        scale = weights
    else:
        log_q = z - state["lse"].double()[:, None]
        scale = weights * state["dloss"].double()
    row = torch.arange(rows, device=z.device)[:, None].expand_as(p)
    grad = log_q.exp()
    grad.index_put_((row[valid], state["index"][valid]), -p[valid], accumulate=True)
    grad *= (scale * case["temperature"])[:, None]
    if kind == "distill_backward":
        return grad
    picked = log_q[row, state["index"].clamp(min=0)]
    loss = (p * (log_p.masked_fill(~valid, 0.0) - picked)).sum(1)
    return weights * case["temperature"] ** 2 * loss, grad


def _exact_sample(state):
    """Row by row in numpy."""
    case = state["case"]
    rows, classes = case["rows"], case["classes"]
    logits = state["logits"].float().cpu().numpy().astype(np.float64)
    uniform = state["uniform"].cpu().numpy().astype(np.float64)
    setting = {k: (v.cpu().numpy() if torch.is_tensor(v) else np.full(rows, v)) for k, v in state["settings"].items()}
    tokens, log_probs = np.empty(rows, dtype=np.int64), np.empty(rows)
    for r in range(rows):
        t, p, least = (float(setting[k][r]) for k in ("temperature", "top_p", "min_p"))
        k = int(setting["top_k"][r])
        w = np.exp((logits[r] - logits[r].max()) / t)
        keep = np.ones(classes, dtype=bool)
        if 0 < k < classes or p < 1:
            order = np.argsort(-logits[r], kind="stable")
            if 0 < k < classes:
                keep[order[k:]] = False
                order = order[:k]
            if p < 1:
                mass = np.concatenate(([0.0], np.cumsum(w[order])))
                dropped = mass[:-1] >= p * mass[-1]
                dropped[0] = False
                keep[order[dropped]] = False
        keep &= w >= min(least, 1.0)
        w = np.where(keep, w, 0.0)
        reached = np.cumsum(w)
        tokens[r] = min(int(np.searchsorted(reached, uniform[r] * reached[-1], side="right")), classes - 1)
        log_probs[r] = math.log(w[tokens[r]] / reached[-1])
    return torch.from_numpy(tokens), torch.from_numpy(log_probs)
