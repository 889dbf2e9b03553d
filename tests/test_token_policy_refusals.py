"""What the token-policy operators refuse: on the CPU, before anything is launched."""

import math

import pytest
import torch

from robolearn_amd import _native
from robolearn_amd import kernels as K

P = 4096  # an aligned address that no refused call reads
FORWARD = dict(type=1, rows=4, inputs=16, hidden=8, activation=0, x=P, ldx=16, w=2 * P, h=3 * P, ld_h=8, workspace=4 * P,
               bytes=1 << 20, stream=None)
BACKWARD = dict(type=1, rows=4, inputs=16, hidden=8, activation=0, x=P, ldx=16, w=2 * P, dh=3 * P, ld_dh=8, dx=4 * P,
                ld_dx=16, dw=5 * P, dw_fp32=0, workspace=6 * P, bytes=1 << 20, stream=None)
DISTILL = dict(logits=P, type=1, ld=100, teacher=2 * P, teacher_type=0, index=3 * P, bits=64, weights=None, rows=4,
               classes=100, entries=8, temperature=1.0, loss=4 * P, lse=None, dlogits=5 * P, ldd=100, scale=1.0, stream=None)
GRADIENT = dict(logits=P, type=1, ld=100, teacher=2 * P, teacher_type=0, index=3 * P, bits=64, weights=None, lse=6 * P,
                dloss=4 * P, rows=4, classes=100, entries=8, temperature=1.0, dlogits=5 * P, ldd=100, stream=None)
SAMPLE = dict(logits=P, type=1, ld=100, rows=4, classes=100, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, temperatures=None,
              top_ks=None, top_ps=None, min_ps=None, uniform=2 * P, tokens=3 * P, log_probs=None, stream=None)


def refused(name, arguments, match, **changes):
    with pytest.raises(RuntimeError, match=match):
        _native.call(name, *{**arguments, **changes}.values())


@pytest.mark.parametrize("changes,match", [
    (dict(type=2), "type"), (dict(rows=-1), "rows"), (dict(rows=(1 << 24) + 1), "rows"), (dict(inputs=0), "inputs"),
    (dict(hidden=0), "hidden"), (dict(inputs=1 << 17, hidden=1 << 16), "2\\^31"), (dict(activation=3), "activation"),
    (dict(activation=-1), "activation"), (dict(x=None), "nonnull"), (dict(w=None), "nonnull"), (dict(h=None), "nonnull"),
    (dict(workspace=None), "workspace"), (dict(bytes=8), "workspace"), (dict(workspace=P + 8), "workspace"),
    (dict(ldx=15), "overlap"), (dict(ld_h=7), "overlap"), (dict(x=P + 1), "aligned"), (dict(h=P + 1), "aligned"),
    (dict(h=P), "overlaps an input"), (dict(h=P + 126), "overlaps an input"), (dict(h=2 * P + 510), "overlaps an input"),
    (dict(workspace=2 * P), "overlaps an input"), (dict(workspace=3 * P), "overlap")])
def test_gated_forward_refuses(changes, match):
    refused("rl_gated_forward", FORWARD, match, **changes)


@pytest.mark.parametrize("changes,match", [
    (dict(dx=None, dw=None), "output"), (dict(dh=None), "nonnull"), (dict(ld_dh=7), "overlap"), (dict(ld_dx=15), "overlap"),
    (dict(dw=P + 1), "aligned"), (dict(dw=P + 2, dw_fp32=1), "aligned"), (dict(bytes=64), "workspace"),
    (dict(type=0, x=P + 2), "aligned"), (dict(dx=P), "overlaps an input"), (dict(dx=3 * P), "overlaps an input"),
    (dict(dw=2 * P), "overlaps an input"), (dict(dw=4 * P), "overlap"), (dict(workspace=5 * P), "overlap")])
def test_gated_backward_refuses(changes, match):
    refused("rl_gated_backward", BACKWARD, match, **changes)


@pytest.mark.parametrize("arguments,name", [(DISTILL, "rl_distill_forward"), (GRADIENT, "rl_distill_backward")])
@pytest.mark.parametrize("changes,match", [
    (dict(type=2), "type"), (dict(teacher_type=5), "type"), (dict(bits=16), "32 or 64"), (dict(rows=-1), "rows"),
    (dict(classes=0), "classes"), (dict(classes=(1 << 24) + 1), "classes"), (dict(entries=0), "entries"),
    (dict(entries=1025), "entries"), (dict(temperature=0.0), "temperature"), (dict(temperature=-1.0), "temperature"),
    (dict(temperature=math.inf), "temperature"), (dict(temperature=math.nan), "temperature"), (dict(logits=None), "nonnull"),
    (dict(teacher=None), "nonnull"), (dict(index=None), "nonnull"), (dict(ld=99), "overlap"), (dict(ldd=99), "overlap"),
    (dict(logits=P + 1), "aligned"), (dict(index=P + 4), "aligned"), (dict(dlogits=P + 2), "place"),
    (dict(rows=1 << 40, dlogits=1 << 60), "Too many rows"),
    (dict(dlogits=P, ldd=101), "place")])
def test_distill_refuses(arguments, name, changes, match):
    refused(name, arguments, match, **changes)


def test_distill_refuses_missing_outputs():
    refused("rl_distill_forward", DISTILL, "loss_rows", loss=None)
    refused("rl_distill_forward", DISTILL, "scale", scale=math.nan)
    refused("rl_distill_backward", GRADIENT, "lse", lse=None)
    refused("rl_distill_backward", GRADIENT, "lse", dloss=None)
    refused("rl_distill_backward", GRADIENT, "lse", dlogits=None)


@pytest.mark.parametrize("changes,match", [
    (dict(type=2), "type"), (dict(rows=-1), "rows"), (dict(classes=0), "classes"), (dict(classes=(1 << 20) + 1), "classes"),
    (dict(logits=None), "nonnull"), (dict(uniform=None), "nonnull"), (dict(tokens=None), "nonnull"), (dict(ld=99), "overlap"),
    (dict(logits=P + 1), "aligned"), (dict(rows=1 << 40), "Too many rows"), (dict(temperature=-0.5), "temperature"), (dict(temperature=math.inf), "temperature"),
    (dict(temperature=math.nan), "temperature"), (dict(top_p=math.nan), "top_p"), (dict(min_p=math.nan), "min_p")])
def test_sample_refuses(changes, match):
    refused("rl_categorical_sample", SAMPLE, match, **changes)


def test_workspace_sizes():
    assert K.gated_workspace(0, 8, 8, torch.bfloat16) == 0
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        assert 0 < K.gated_workspace(5, 9, 7, dtype) <= K.gated_workspace(5, 9, 7, dtype, backward=True)
    for arguments in ((-1, 8, 8, torch.float32), (1, 0, 8, torch.float32), (1, 8, 8, torch.float64)):
        with pytest.raises(ValueError):
            K.gated_workspace(*arguments)


X, W, H = torch.zeros(4, 16), torch.zeros(2, 8, 16), torch.zeros(4, 8)
Z, T, I = torch.zeros(4, 100), torch.zeros(4, 8), torch.zeros(4, 8, dtype=torch.int64)
V, N = torch.zeros(4), torch.zeros(4, dtype=torch.int64)


@pytest.mark.parametrize("call", [
    lambda: K.gated_forward(X.double(), W, H), lambda: K.gated_forward(X, W.half(), H), lambda: K.gated_forward(X, W[:1], H),
    lambda: K.gated_forward(X, W[:, :, :8], H), lambda: K.gated_forward(X, W, H[:, :7]), lambda: K.gated_forward(X, W, H.half()),
    lambda: K.gated_forward(X.t().contiguous().t(), W, H), lambda: K.gated_forward(X[:1].expand(4, 16), W, H),
    lambda: K.gated_forward(X, W.transpose(1, 2).contiguous().transpose(1, 2), H),
    lambda: K.gated_forward(X, W, H, activation="tanh"), lambda: K.gated_forward(X[0], W, H),
    lambda: K.gated_backward(X, W, H[:3], X.clone(), None), lambda: K.gated_backward(X, W, H, X[:, :8], None),
    lambda: K.gated_backward(X, W, H, None, W.half()), lambda: K.gated_backward(X, W, H, None, W[:, :4]),
    lambda: K.distill_forward(Z, T[:3], I, V), lambda: K.distill_forward(Z, T, I[:, :4], V),
    lambda: K.distill_forward(Z, T, I.float(), V), lambda: K.distill_forward(Z, T, I, V[:3]),
    lambda: K.distill_forward(Z, T, I, V, temperature=0.0), lambda: K.distill_forward(Z, T, I, V, weights=V[:2]),
    lambda: K.distill_forward(Z, T, I, V, dlogits=Z.half()), lambda: K.distill_forward(Z, T, I, V, lse=V.double()),
    lambda: K.distill_forward(Z, T.t().contiguous().t(), I, V), lambda: K.distill_forward(Z.int(), T, I, V),
    lambda: K.distill_backward(Z, T, I, V, V[:1], Z.clone()), lambda: K.distill_backward(Z, T, I, V, V, Z[:, :50]),
    lambda: K.categorical_sample(Z, V[:2], N), lambda: K.categorical_sample(Z, V, N.int()),
    lambda: K.categorical_sample(Z[0], V, N), lambda: K.categorical_sample(Z, V, N, log_probs=V.half()),
    lambda: K.categorical_sample(Z, V, N, temperature=V[:2]), lambda: K.categorical_sample(Z, V, N, top_k=V),
    lambda: K.categorical_sample(Z, V.double(), N), lambda: K.categorical_sample(Z.t().contiguous().t(), V, N),
    # on the CPU
    lambda: K.gated_forward(X, W, H), lambda: K.distill_forward(Z, T, I, V), lambda: K.categorical_sample(Z, V, N)])
def test_wrappers_refuse(call):
    with pytest.raises(ValueError):
        call()
