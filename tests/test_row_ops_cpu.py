"""Refusals of the language-model row operators, which come before any device
is touched: through torch_ops with host tensors, and at the C entry points."""
import ctypes

import pytest
import torch

from hephaestus_b200 import InvalidConfiguration
from hephaestus_b200 import _native as N
from hephaestus_b200 import torch_ops as T


def refused(message, call, *args, **kw):
    with pytest.raises(InvalidConfiguration) as e:
        call(*args, **kw)
    assert message in e.value.message, e.value.message


X = torch.zeros(4, 64)


def test_norm_refusals():
    refused("f32, bf16 or f16", T.rms_norm, X.double())
    refused("rows and columns", T.rms_norm, X[0])
    refused("adjacent columns", T.rms_norm, X.t())
    refused("equal distances", T.rms_norm, torch.zeros(3, 4, 8).transpose(0, 1))
    refused("residual has shape", T.rms_norm, X, residual=X[:2])
    refused("residual must be", T.rms_norm, X, residual=X.half())
    refused("weight must be", T.rms_norm, X, torch.zeros(64, dtype=torch.float16))
    refused("vector of 64", T.rms_norm, X, torch.zeros(63))
    refused("vector of 64", T.rms_norm, X, torch.zeros(128)[::2])
    refused("detach it", T.rms_norm, X.clone().requires_grad_())
    refused("detach it", T.rms_norm, X, torch.zeros(64, requires_grad=True))
    refused("power of two", T.rms_norm_fp8, X, group=24)
    refused("power of two", T.rms_norm_fp8, X, group=8)
    refused("dsum must be", T.rms_norm_backward, X, X, dsum=X.half())
    refused("dy has shape", T.rms_norm_backward, X[:1], X)
    refused("s must have", T.rms_norm_backward, X.t(), X.t())
    refused("must be a torch tensor", T.rms_norm, None)
    refused("plain values", T.rms_norm, torch._neg_view(X))
    refused("plain values", T.rms_norm, X, torch._neg_view(X[0]))
    refused("plain values", T.rms_norm, X.to_sparse())
    with torch.no_grad():  # nothing is recorded: the device is asked for next
        refused("needs CUDA tensors", T.rms_norm, X, torch.zeros(64, requires_grad=True))
    refused("needs CUDA tensors", T.rms_norm, X, torch.zeros(64))


def test_route_refusals():
    refused("unknown routing score", T.route_experts, X, 2, score="relu")
    refused("chooses 1 to 32", T.route_experts, X, 0)
    refused("chooses 1 to 32", T.route_experts, X, 33)
    refused("chooses 1 to 32", T.route_experts, X[:, :4], 5)
    refused("chooses 1 to 32", T.route_experts, torch.zeros(1, 1025), 2)
    refused("vector of 64", T.route_experts, X, 2, bias=torch.zeros(4))
    refused("bias must be", T.route_experts, X, 2, bias=torch.zeros(64).double())
    refused("detach it", T.route_experts, X.clone().requires_grad_(), 2)
    g, p = torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.int32)
    refused("dweights has shape", T.route_experts_backward, g[:3], X, p)
    refused("experts must be", T.route_experts_backward, g, X, p.long())
    refused("leading dimensions", T.route_experts_backward, g, X, p[0])
    refused("needs CUDA tensors", T.route_experts_backward, g, X, p)


def test_order_and_sample_refusals():
    p = torch.zeros(4, 2, dtype=torch.int32)
    refused("torch.int32", T.expert_order, p.long(), 4)
    refused("contiguous", T.expert_order, p.t(), 4)
    refused("1 to 1024", T.expert_order, p, 0)
    refused("1 to 1024", T.expert_order, p, 1025)
    refused("needs CUDA tensors", T.expert_order, p, 4)
    u = torch.zeros(4)
    refused("[rows, vocabulary]", T.sample_tokens, torch.zeros(2, 2, 8), u)
    refused("[rows, vocabulary]", T.sample_tokens, torch.zeros(4, 0), u)
    refused("vector of 4", T.sample_tokens, X, u[:3])
    refused("uniform must be", T.sample_tokens, X, u.double())
    refused("top_k must be", T.sample_tokens, X, u, top_k=torch.zeros(4))
    refused("vector of 4", T.sample_tokens, X, u, temperature=torch.zeros(1))
    refused("needs CUDA tensors", T.sample_tokens, X, u)


# At the C entry points: addresses that nothing reads, since every call is refused.
A, B, C, D = 0x1000000, 0x2000000, 0x3000000, 0x4000000


def c_refused(message, name, *args):
    assert getattr(N.lib, name)(*args) == N.INVALID_CONFIGURATION
    assert message in N.last_error(), N.last_error()


def norm_args(**kw):
    a = dict(ordinal=0, dtype=N.ROW_F32, x=A, xs=64, res=None, rs=0, w=None, wd=N.ROW_F32, eps=1e-6, rows=4, cols=64, y=B,
             sum=None, stream=None) | kw
    return list(a.values())


@pytest.mark.parametrize("message,kw", [
    ("f32, bf16 or f16", dict(dtype=3)), ("f32, bf16 or f16", dict(dtype=-1)), ("weight of the rows' type", dict(w=C, wd=N.ROW_F16)),
    ("finite eps", dict(eps=-1.0)), ("finite eps", dict(eps=float("nan"))), ("finite eps", dict(eps=float("inf"))),
    ("no columns", dict(cols=0)), ("out of range", dict(rows=1 << 31)), ("out of range", dict(cols=(1 << 24) + 1)),
    ("x is null", dict(x=None)), ("y is null", dict(y=None)), ("not aligned", dict(x=A + 2)), ("negative row stride", dict(xs=-64)),
    ("row stride out of range", dict(xs=1 << 62)), ("only with, a residual", dict(res=C)), ("only with, a residual", dict(sum=C)),
    ("alias its inputs", dict(y=A)), ("alias its inputs", dict(y=A + 3 * 256)), ("alias its inputs", dict(w=B + 128)),
    ("alias one another", dict(res=C, rs=64, sum=B + 4)),
])
def test_c_norm_refusals(message, kw):
    c_refused(message, "heph_rms_norm", *norm_args(**kw))


def test_c_fp8_refusals():
    def args(group=0, cols=64, q=B, scales=C, res=None, sum_=None):
        return [0, N.ROW_F32, A, cols, res, cols, None, N.ROW_F32, 1e-6, 4, cols, group, q, scales, sum_, None]
    c_refused("power of two", "heph_rms_norm_fp8", *args(group=48))
    c_refused("power of two", "heph_rms_norm_fp8", *args(group=8))
    c_refused("at most 8192 groups", "heph_rms_norm_fp8", *args(group=16, cols=16 * 8193))
    c_refused("scales is null", "heph_rms_norm_fp8", *args(scales=None))
    c_refused("alias one another", "heph_rms_norm_fp8", *args(scales=B + 4))
    c_refused("only with, a residual", "heph_rms_norm_fp8", *args(res=D))


def test_c_backward_refusals():
    def args(dw=D, w=C, work=0x5000000, size=1 << 20):
        return [0, N.ROW_F32, A, 64, A, 64, None, 0, w, N.ROW_F32, 1e-6, 4, 64, B, dw, work, size, None]
    c_refused("no weight to differentiate", "heph_rms_norm_backward", *args(w=None))
    c_refused("alias its inputs", "heph_rms_norm_backward", *args(work=A))
    c_refused("alias one another", "heph_rms_norm_backward", *args(work=B + 16))
    c_refused("aligned to 16", "heph_rms_norm_backward", *args(work=0x5000004))
    c_refused("null output", "heph_rms_norm_backward_workspace", 0, 4, 64, None)
    need = ctypes.c_uint64()
    c_refused("out of range", "heph_rms_norm_backward_workspace", 0, 1 << 32, 64, ctypes.byref(need))


def test_c_route_refusals():
    def args(experts=64, k=4, score=0, groups=1, kept=1, top=2, bias=None, weights=B, picks=C, dtype=N.ROW_F32):
        return [0, dtype, A, experts, bias, 4, experts, k, score, groups, kept, top, 1, 1.0, weights, picks, None]
    name = "heph_route_experts"
    c_refused("f32, bf16 or f16", name, *args(dtype=9))
    c_refused("1 to 1024 experts", name, *args(experts=1025))
    c_refused("1 to 1024 experts", name, *args(experts=0))
    c_refused("chooses 1 to 32", name, *args(k=0))
    c_refused("chooses 1 to 32", name, *args(experts=3, k=4))
    c_refused("unknown routing score", name, *args(score=2))
    c_refused("groups of equal size", name, *args(groups=7))
    c_refused("groups of equal size", name, *args(groups=0))
    c_refused("groups of equal size", name, *args(groups=64))
    c_refused("keeps 1 to all", name, *args(groups=8, kept=9))
    c_refused("keeps 1 to all", name, *args(groups=8, kept=0))
    c_refused("one or two best", name, *args(top=3))
    c_refused("cannot choose 9", name, *args(groups=8, kept=1, k=9))
    c_refused("picks is null", name, *args(picks=None))
    c_refused("alias one another", name, *args(picks=B + 8))
    c_refused("alias its inputs", name, *args(weights=A))
    back = [0, N.ROW_F32, B, 4, A, 64, C, 4, 4, 64, 4, 0, 1, 1.0, D, None]
    for at, value, message in ((1, 5, "f32, bf16"), (10, 0, "chooses"), (11, 7, "unknown"), (2, None, "dweights is null"),
                               (14, A, "alias its inputs"), (7, -4, "negative")):
        c_refused(message, "heph_route_experts_backward", *(back[:at] + [value] + back[at + 1:]))


def test_c_order_refusals():
    good = [0, A, 100, 8, B, C, D, None, 0, None]
    for at, value, message in ((3, 0, "1 to 1024"), (3, 1025, "1 to 1024"), (2, 1 << 31, "out of range"), (1, None, "picks is null"),
                               (4, None, "offsets is null"), (5, None, "order is null"), (6, None, "slot is null"),
                               (5, A, "alias its inputs"), (6, C + 4, "alias one another"), (4, B + 2, "not aligned"), (2, 200000, "needs a workspace of 3136 bytes")):
        c_refused(message, "heph_expert_order", *(good[:at] + [value] + good[at + 1:]))
    c_refused("not aligned to 16", "heph_expert_order", *(good[:7] + [0x5000008, 64, None]))
    need = ctypes.c_uint64()
    c_refused("null output", "heph_expert_order_workspace", 4, 4, None)
    c_refused("out of range", "heph_expert_order_workspace", 1 << 31, 4, ctypes.byref(need))


def test_c_sample_refusals():
    def args(**kw):
        a = dict(ordinal=0, dtype=N.ROW_F32, logits=A, stride=1000, rows=4, vocab=1000, u=B, tp=None, t=1.0, kp=None, k=0, pp=None,
                 p=1.0, mp=None, m=0.0, tokens=C, probs=D, stream=None) | kw
        return list(a.values())
    nan = float("nan")
    for kw, message in ((dict(dtype=4), "f32, bf16"), (dict(vocab=0), "vocabulary"), (dict(vocab=(1 << 26) + 1), "vocabulary"),
                        (dict(rows=1 << 31), "rows out of range"), (dict(t=-0.1), "temperature"), (dict(t=nan), "temperature"),
                        (dict(t=float("inf")), "temperature"), (dict(k=-1), "top_k"), (dict(p=1.5), "top_p"), (dict(p=nan), "top_p"),
                        (dict(m=-0.5), "min_p"), (dict(m=2.0), "min_p"), (dict(u=None), "uniform is null"),
                        (dict(tokens=None), "tokens is null"), (dict(probs=None), "probs is null"),
                        (dict(tokens=C + 4), "not aligned"), (dict(tokens=A), "alias its inputs"), (dict(probs=B), "alias its inputs"),
                        (dict(probs=C + 8), "alias one another"), (dict(kp=D), "alias its inputs")):
        c_refused(message, "heph_sample_tokens", *args(**kw))


def test_the_library_builds_without_torch(monkeypatch):
    from hephaestus_b200 import build
    monkeypatch.setattr(build.importlib.util, "find_spec", lambda name: None)
    assert build.build_torch_module() is None


def test_an_empty_call_needs_no_device():
    """Nothing to do is done without touching a device (none is here in the CPU suite)."""
    assert N.lib.heph_rms_norm(*norm_args(rows=0, x=None, y=None)) == N.OK


def test_a_call_without_a_gpu_is_an_error():
    if torch.cuda.is_available():
        pytest.skip("a GPU is visible")
    assert N.lib.heph_rms_norm(*norm_args()) == N.DEVICE_UNAVAILABLE
