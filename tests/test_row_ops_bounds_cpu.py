"""Refusals of the language-model row operators at the bounds of their arguments' types, which come
before any device is touched: with tensors of no memory, or on the host."""
import pytest
import torch

from hephaestus_b200 import InvalidConfiguration
from hephaestus_b200 import _native as N
from hephaestus_b200 import torch_ops as T


def refused(message, call, *args, **kw):
    with pytest.raises(InvalidConfiguration) as e:
        call(*args, **kw)
    assert message in e.value.message, e.value.message


def test_sizes_past_32_bits():
    """No size is taken for what its low 32 bits say."""
    def wide(cols, dtype):
        return torch.empty(1, cols, dtype=dtype, device="meta")
    past = 2 ** 32 + 8
    g, p = torch.zeros(1, 2), torch.zeros(1, 2, dtype=torch.int32)
    refused(f"2 of {past}", T.route_experts_backward, g, wide(past, torch.bfloat16), p)
    refused(f"{past} of 8", T.route_experts_backward, wide(past, torch.float32), torch.zeros(1, 8), wide(past, torch.int32))
    refused("chooses 1 to 32", T.route_experts_backward, torch.zeros(1, 0), torch.zeros(1, 8), p[:, :0])
    refused(f"2 of {past}", T.route_experts, wide(past, torch.bfloat16), 2)
    refused("1 to 1024", T.expert_order, p, past)
    refused("[rows, vocabulary]", T.sample_tokens, wide(past, torch.bfloat16), torch.zeros(1))


def test_forward_mode_tensors_are_refused():
    """A tangent is not dropped in silence."""
    from torch.autograd import forward_ad
    x, w = torch.ones(4, 64), torch.ones(64)
    p = torch.zeros(4, 2, dtype=torch.int32)
    with forward_ad.dual_level():
        d, dw = forward_ad.make_dual(x, x), forward_ad.make_dual(w, w)
        du = forward_ad.make_dual(torch.zeros(4), torch.ones(4))
        dg = forward_ad.make_dual(x[:, :2].clone(), x[:, :2].clone())
        for call, args, kw in ((T.rms_norm, (d,), {}), (T.rms_norm, (x, dw), {}), (T.rms_norm, (x,), dict(residual=d)),
                               (T.rms_norm_fp8, (d,), {}), (T.rms_norm_backward, (d, x), {}), (T.rms_norm_backward, (x, d), {}),
                               (T.rms_norm_backward, (x, x), dict(dsum=d)), (T.route_experts, (d, 2), {}),
                               (T.route_experts, (x, 2), dict(bias=dw)), (T.route_experts_backward, (dg, x, p), {}),
                               (T.route_experts_backward, (x[:, :2], d, p), {}), (T.sample_tokens, (d, torch.zeros(4)), {}),
                               (T.sample_tokens, (x, du), {}), (T.sample_tokens, (x, torch.zeros(4)), dict(temperature=du))):
            refused("has a tangent", call, *args, **kw)
            with torch.no_grad():
                refused("has a tangent", call, *args, **kw)
        refused("needs CUDA tensors", T.rms_norm, forward_ad.unpack_dual(d).primal)
    refused("needs CUDA tensors", T.rms_norm, d)  # outside its level it is the primal


@pytest.mark.parametrize("eps,good", [(0.0, True), (1.2e-38, True), (3.4e38, True), (1e-39, False), (1e-60, False), (3.5e38, False),
                                      (1e300, False)])
def test_an_eps_that_32_bits_do_not_hold(eps, good):
    """As 32 bits a smaller one is 0, and a row of zeros 0 / 0; a larger one is infinite."""
    a = 0x1000000  # an address that nothing reads: without rows nothing is done
    norm = N.lib.heph_rms_norm(0, N.ROW_F32, a, 64, None, 0, None, N.ROW_F32, eps, 0, 64, 2 * a, None, None)
    fp8 = N.lib.heph_rms_norm_fp8(0, N.ROW_F32, a, 64, None, 0, None, N.ROW_F32, eps, 0, 64, 0, 2 * a, 3 * a, None, None)
    grad = N.lib.heph_rms_norm_backward(0, N.ROW_F32, a, 64, a, 64, None, 0, None, N.ROW_F32, eps, 0, 64, 2 * a, None, None, 0, None)
    assert {norm, fp8, grad} == {N.OK if good else N.INVALID_CONFIGURATION}
    if not good:
        assert "normal f32 numbers" in N.last_error()
