"""torch boundary: the module-level functions of the reference's Python
bindings (``sum``, ``min``, ``max``, ``mean``, ``sum_axis``, ``mean_axis``,
``min_axis``, ``max_axis``, ``norm_l1``, ``norm_l2``, ``norm_max``,
``cumsum`` — crates/hephaestus-python/src/reduction.rs:112-367, scan.rs:13)
over CUDA torch tensors, plus ``argmax_axis`` / ``argmin_axis`` / ``cumprod``
/ exclusive scans [EXT] and the row operators of language models [EXT]
(``rms_norm``, ``rms_norm_fp8``, ``rms_norm_backward``, ``route_experts``,
``route_experts_backward``, ``expert_order``, ``sample_tokens``).

The tensors' memory is wrapped, not copied (``heph_buffer_wrap``); the work is
enqueued on torch's current stream and results are returned as new tensors
allocated by torch, so these calls compose with ordinary torch code.  Strided
(non-contiguous) tensors are passed as strided views.
"""
from __future__ import annotations

import builtins
import ctypes

import torch

from . import _native as N
from .core import CudaBuffer, CudaDevice, InvalidConfiguration, Layout, StridedView, check

try:
    from . import _torch_rows
except ImportError as e:  # all but the row operators needs the library alone

    class _Absent:
        why = str(e)

        def __getattr__(self, name):
            raise ImportError(f"{name} needs hephaestus_b200/_torch_rows.so, which build.py makes for the installed torch: {self.why}")

    _torch_rows = _Absent()

_TORCH_DTYPES = {torch.float32: N.F32, torch.float64: N.F64, torch.int32: N.I32, torch.int64: N.I64}
if hasattr(torch, "uint32"):
    _TORCH_DTYPES[torch.uint32] = N.U32
_devices: dict[int, CudaDevice] = {}


def _device(t: torch.Tensor) -> CudaDevice:
    if not t.is_cuda:
        raise InvalidConfiguration("hephaestus_b200.torch_ops needs CUDA tensors")
    idx = t.device.index if t.device.index is not None else torch.cuda.current_device()
    if idx not in _devices:
        _devices[idx] = CudaDevice(idx)
    return _devices[idx]


def _view(t: torch.Tensor) -> StridedView:
    """Wrap a tensor's memory as a buffer + layout (no copy)."""
    if t.dtype not in _TORCH_DTYPES:
        raise InvalidConfiguration(f"unsupported tensor dtype {t.dtype}")
    dev = _device(t)
    span = 1 + builtins.sum((s - 1) * st for s, st in zip(t.shape, t.stride())) if t.numel() else 0
    h = ctypes.c_void_p()
    check(N.lib.heph_buffer_wrap(dev.handle, _TORCH_DTYPES[t.dtype], ctypes.c_void_p(t.data_ptr()), span,
                                 ctypes.byref(h)))
    buf = CudaBuffer(dev, h.value)
    buf._keep = t  # the tensor outlives the wrapper
    shape = list(t.shape) or [1]
    strides = list(t.stride()) or [1]
    return StridedView(buf, Layout.try_new(shape, strides, 0))


def _stream() -> int:
    """torch's current stream.  Its default stream is the legacy one, whose own
    handle (cudaStreamLegacy) is passed: a null stream means the device's."""
    return torch.cuda.current_stream().cuda_stream or 1


def _full(op_code: int, t: torch.Tensor) -> torch.Tensor:
    out = torch.empty(1, dtype=t.dtype, device=t.device)
    iv, ov = _view(t), _view(out)
    check(N.lib.heph_reduce_full(iv.buffer.device.handle, op_code, iv.buffer.handle, ctypes.byref(iv.layout.native()),
                                 ov.buffer.handle, ctypes.byref(ov.layout.native()), ctypes.c_void_p(_stream())))
    return out.reshape(())


def sum(t: torch.Tensor) -> torch.Tensor:  # noqa: A001 - reference name
    return _full(N.SUM, t)


def prod(t: torch.Tensor) -> torch.Tensor:
    return _full(N.PROD, t)


def min(t: torch.Tensor) -> torch.Tensor:  # noqa: A001
    return _full(N.MIN, t)


def max(t: torch.Tensor) -> torch.Tensor:  # noqa: A001
    return _full(N.MAX, t)


def mean(t: torch.Tensor) -> torch.Tensor:
    s = sum(t)
    return s / t.numel() if t.dtype.is_floating_point else torch.div(s, t.numel(), rounding_mode="trunc")


def _axis(op_code: int, t: torch.Tensor, axis: int) -> torch.Tensor:
    if t.dim() != 2:
        raise InvalidConfiguration("axis reductions take rank-2 tensors")
    shape = list(t.shape)
    shape[axis] = 1
    out = torch.empty(shape, dtype=t.dtype, device=t.device)
    iv, ov = _view(t), _view(out)
    check(N.lib.heph_reduce_axis(iv.buffer.device.handle, op_code, iv.buffer.handle, ctypes.byref(iv.layout.native()),
                                 int(axis), ov.buffer.handle, ctypes.byref(ov.layout.native()),
                                 ctypes.c_void_p(_stream())))
    return out


def sum_axis(t, axis):
    return _axis(N.SUM, t, axis)


def mean_axis(t, axis):
    return _axis(N.MEAN, t, axis)


def min_axis(t, axis):
    return _axis(N.MIN, t, axis)


def max_axis(t, axis):
    return _axis(N.MAX, t, axis)


def prod_axis(t, axis):
    return _axis(N.PROD, t, axis)


def _arg(op_code: int, t: torch.Tensor, axis: int):
    if t.dim() != 2:
        raise InvalidConfiguration("arg-reductions take rank-2 tensors")
    shape = list(t.shape)
    shape[axis] = 1
    vals = torch.empty(shape, dtype=t.dtype, device=t.device)
    idx = torch.empty(shape, dtype=torch.int32, device=t.device)
    iv, vv = _view(t), _view(vals)
    h = ctypes.c_void_p()
    check(N.lib.heph_buffer_wrap(iv.buffer.device.handle, N.U32, ctypes.c_void_p(idx.data_ptr()), idx.numel(),
                                 ctypes.byref(h)))
    ib = CudaBuffer(iv.buffer.device, h.value)
    il = Layout.c_contiguous(shape)
    check(N.lib.heph_arg_reduce_axis(iv.buffer.device.handle, op_code, iv.buffer.handle,
                                     ctypes.byref(iv.layout.native()), int(axis), vv.buffer.handle,
                                     ctypes.byref(vv.layout.native()), ib.handle, ctypes.byref(il.native()),
                                     ctypes.c_void_p(_stream())))
    return vals, idx.to(torch.int64)


def argmax_axis(t, axis):
    """[EXT] (values, indices) of the maxima along `axis`; lowest index wins ties."""
    return _arg(N.MAX, t, axis)


def argmin_axis(t, axis):
    """[EXT] (values, indices) of the minima along `axis`; lowest index wins ties."""
    return _arg(N.MIN, t, axis)


def _scan(op_code: int, t: torch.Tensor, axis: int, reverse: bool, exclusive: bool) -> torch.Tensor:
    if t.dim() not in (1, 2):
        raise InvalidConfiguration("scans take rank-1 or rank-2 tensors")
    out = torch.empty(t.shape, dtype=t.dtype, device=t.device)
    iv, ov = _view(t), _view(out)
    check(N.lib.heph_scan_axis(iv.buffer.device.handle, op_code, N.REVERSE if reverse else N.FORWARD,
                               int(bool(exclusive)), iv.buffer.handle, ctypes.byref(iv.layout.native()), int(axis),
                               ov.buffer.handle, ctypes.byref(ov.layout.native()), ctypes.c_void_p(_stream())))
    return out


def cumsum(t, axis=0, reverse=False, exclusive=False):
    return _scan(N.SUM, t, axis, reverse, exclusive)


def cumprod(t, axis=0, reverse=False, exclusive=False):
    return _scan(N.PROD, t, axis, reverse, exclusive)


def _map(map_kind: int, a: torch.Tensor, b: torch.Tensor | None = None) -> torch.Tensor:
    out = torch.empty(1, dtype=a.dtype, device=a.device)
    av, ov = _view(a), _view(out)
    bv = _view(b) if b is not None else None
    check(N.lib.heph_map_reduce_full(av.buffer.device.handle, map_kind, av.buffer.handle,
                                     ctypes.byref(av.layout.native()),
                                     bv.buffer.handle if bv is not None else None,
                                     ctypes.byref(bv.layout.native()) if bv is not None else None,
                                     ov.buffer.handle, ctypes.byref(ov.layout.native()),
                                     ctypes.c_void_p(_stream())))
    return out.reshape(())


def dot(a, b):
    return _map(N.MAP_DOT, a, b)


def norm_l1(t):
    return _map(N.MAP_NORM_L1, t)


def norm_l2(t):
    return _map(N.MAP_NORM_L2, t)


def norm_max(t):
    return _map(N.MAP_NORM_MAX, t)


# --------------------------------------------- language-model row operators [EXT]
#
# Over the rows of a matrix whose columns are adjacent (rows may be any
# distance apart; leading dimensions that form one are taken together).  They
# run on the tensors' own device and that device's current torch stream, write
# new contiguous tensors, and may be captured into a graph.  There is no
# autograd in this module: gradients are calls of their own, and a tensor that
# asks for one is refused while gradients are recorded.  The checks and the
# calls are in csrc/torch_rows.cpp.


def rms_norm(x, weight=None, eps=1e-6, *, residual=None):
    """[EXT] y = weight * s / sqrt(mean(s^2) + eps) over the last dimension, s = x (+ residual).

    x: f32, bf16 or f16; weight: of x's type or f32 (None: ones); eps: 0 or a normal f32 number.
    Returns y, or (y, s) with a residual; both in x's type, each rounded once."""
    return _torch_rows.rms_norm(x, weight, eps, residual)


def rms_norm_fp8(x, weight=None, eps=1e-6, *, residual=None, group=None):
    """[EXT] rms_norm with an e4m3 result and its scales: y ~ q * scale.

    One scale for a row, or for each `group` adjacent columns (a power of two of 16 or more; the
    last group may be shorter): max(max|y|, 2^-100) / 448.  Returns (q, scales), or (q, scales, s) with
    a residual; scales f32 [..., groups]."""
    return _torch_rows.rms_norm_fp8(x, weight, eps, residual, group)


def rms_norm_backward(dy, s, weight=None, eps=1e-6, *, dsum=None):
    """[EXT] Gradients of rms_norm at s (its x, or the sum that it returned).

    dsum: the gradient that reaches s by other ways (the residual stream), added.  Returns
    (ds, dweight): ds in s's type, the gradient of x and of the residual alike; dweight in the
    weight's type, summed over all rows in a fixed order (None without a weight)."""
    return _torch_rows.rms_norm_backward(dy, s, weight, eps, dsum)


def route_experts(logits, k, *, score="softmax", bias=None, groups=1, groups_kept=1, group_top=2, renormalize=True,
                  scale=1.0):
    """[EXT] The k experts of every row of `logits` [..., experts] and their weights.

    Scores are the logits' softmax or sigmoid; score + bias (f32 [experts]) chooses, the score
    weighs.  With groups > 1 a group of adjacent experts is worth the sum of its group_top (1 or 2)
    best choices, and only the best groups_kept groups stay.  Experts come in falling order, the
    lowest index first among equals.  renormalize divides by the sum of the chosen scores.  Returns
    (weights f32 [..., k], experts i32 [..., k]); an expert whose logit is -inf or NaN is not
    chosen, and where none is left the expert is -1 with weight 0."""
    return _torch_rows.route_experts(logits, k, score, bias, groups, groups_kept, group_top, renormalize, scale)


def route_experts_backward(dweights, logits, experts, *, score="softmax", renormalize=True, scale=1.0):
    """[EXT] Gradient of route_experts' weights by its logits, for the experts that it chose.

    dweights f32 [..., k], experts i32 [..., k] as returned.  Returns dlogits like logits (the bias
    only chooses, so it has no gradient)."""
    return _torch_rows.route_experts_backward(dweights, logits, experts, score, renormalize, scale)


def expert_order(experts, num_experts):
    """[EXT] The routed pairs of `experts` (i32, as route_experts returns it) in the order of experts.

    Returns (offsets i32 [num_experts + 1], order i32 [pairs], slot like experts): the pairs of expert
    e are order[offsets[e]:offsets[e + 1]], as places in the flattened `experts`, in rising order; slot is
    the inverse.  A pair whose expert is outside [0, num_experts) has slot -1, and order is -1 past
    the last pair."""
    return _torch_rows.expert_order(experts, num_experts)


def sample_tokens(logits, uniform, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """[EXT] A token from every row of `logits` [rows, vocabulary], by the numbers `uniform` (f32 [rows], in [0, 1)).

    Weights are exp((l - max) / temperature).  In falling order of the logits (the lowest index first
    among equals) top_k keeps the first k (0: off), top_p of those the ones before which lies less
    than top_p of their mass (1: off), min_p of those the ones of at least min_p of the largest weight
    (0: off).  The token is the first index whose running sum of kept weights exceeds uniform times
    their whole (a weight below 2^-45 of the largest, 2^-39 in the widest vocabularies, counts as none);
    temperature 0 takes the largest.  Each setting is a number or a tensor of one per
    row (f32; top_k i32), where a top_k <= 0, a top_p >= 1, a min_p <= 0 and NaN are off, a top_p <= 0
    leaves the first, a min_p >= 1 those equal to the largest, and a temperature <= 0 or NaN takes the
    largest.  The answer for a row is the same in any batch.  Returns (tokens i64 [rows], probs f32
    [rows]), the probability among the kept ones; a row of nothing but -inf and NaN has token -1."""
    return _torch_rows.sample_tokens(logits, uniform, temperature, top_k, top_p, min_p)
