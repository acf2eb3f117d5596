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
    return torch.cuda.current_stream().cuda_stream


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
# asks for one is refused while gradients are recorded.

_ROW_DTYPES = {torch.float32: N.ROW_F32, torch.bfloat16: N.ROW_BF16, torch.float16: N.ROW_F16}
_ROUTE_SCORES = {"softmax": N.ROUTE_SOFTMAX, "sigmoid": N.ROUTE_SIGMOID}


def _refuse(message: str):
    raise InvalidConfiguration(message)


def _rows(name: str, t: torch.Tensor, shape=None, dtype=None) -> torch.Tensor:
    """`t` as a matrix with adjacent columns (of `shape` and `dtype`, if given)."""
    if dtype is None:
        if t.dtype not in _ROW_DTYPES:
            _refuse(f"{name} must be f32, bf16 or f16, not {t.dtype}")
    elif t.dtype != dtype:
        _refuse(f"{name} must be {dtype}, not {t.dtype}")
    if shape is not None and t.shape != shape:
        _refuse(f"{name} has shape {list(t.shape)}, not {list(shape)}")
    if t.dim() != 2:
        if t.dim() < 2:
            _refuse(f"{name} must have rows and columns")
        try:
            t = t.view(-1, t.shape[-1]) if t.numel() else t.reshape(-1, t.shape[-1] or 1)[:, :t.shape[-1]]
        except RuntimeError:
            _refuse(f"{name} has leading dimensions that do not form rows at equal distances")
    if t.stride(1) != 1 and t.shape[1] > 1:
        _refuse(f"{name} must have adjacent columns")
    if t.requires_grad and torch.is_grad_enabled():
        _refuse(f"{name} asks for a gradient, which these calls do not record: detach it, or use torch.no_grad()")
    return t


def _vector(name: str, t: torch.Tensor, length: int, dtypes) -> torch.Tensor:
    if t.dtype not in dtypes:
        _refuse(f"{name} must be {' or '.join(str(d) for d in dtypes)}, not {t.dtype}")
    if t.dim() != 1 or t.shape[0] != length or (t.stride(0) != 1 and length > 1):
        _refuse(f"{name} must be a vector of {length} adjacent elements")
    if t.requires_grad and torch.is_grad_enabled():
        _refuse(f"{name} asks for a gradient, which these calls do not record: detach it, or use torch.no_grad()")
    return t


def _ordinal(first: torch.Tensor, *others) -> int:
    """The CUDA device that all operands (None: absent) are on."""
    if not first.is_cuda:
        _refuse("hephaestus_b200.torch_ops needs CUDA tensors")
    at = first.get_device()
    for t in others:
        if t is not None and t.get_device() != at:
            _refuse("operands are on different devices")
    return at


def _raw_stream(ordinal: int) -> int:
    """The device's current torch stream; 0 is the legacy default stream, which
    the row operators take as it is."""
    return torch._C._cuda_getCurrentRawStream(ordinal)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _norm_operands(x, weight, residual):
    """Matrix, its columns, the residual as a matrix, and codes of both types."""
    m = _rows("x", x)
    cols = m.shape[1]
    r = None if residual is None else _rows("residual", residual, x.shape, x.dtype)
    code = wcode = _ROW_DTYPES[m.dtype]
    if weight is not None:
        _vector("weight", weight, cols, (m.dtype, torch.float32))
        wcode = _ROW_DTYPES[weight.dtype]
    return m, cols, r, code, wcode


def rms_norm(x, weight=None, eps=1e-6, *, residual=None):
    """[EXT] y = weight * s / sqrt(mean(s^2) + eps) over the last dimension, s = x (+ residual).

    x: f32, bf16 or f16; weight: of x's type or f32 (None: ones).  Returns y, or (y, s) with a
    residual; both in x's type, each rounded once."""
    m, cols, r, code, wcode = _norm_operands(x, weight, residual)
    at = _ordinal(m, r, weight)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    s = None if r is None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    check(N.lib.heph_rms_norm(at, code, m.data_ptr(), m.stride(0), _ptr(r), 0 if r is None else r.stride(0),
                              _ptr(weight), wcode, eps, m.shape[0], cols, y.data_ptr(), _ptr(s), _raw_stream(at)))
    return y if s is None else (y, s)


def rms_norm_fp8(x, weight=None, eps=1e-6, *, residual=None, group=None):
    """[EXT] rms_norm with an e4m3 result and its scales: y ~ q * scale.

    One scale for a row, or for each `group` adjacent columns (a power of two of 16 or more; the
    last group may be shorter): max(max|y|, 2^-100) / 448.  Returns (q, scales), or (q, scales, s) with
    a residual; scales f32 [..., groups]."""
    m, cols, r, code, wcode = _norm_operands(x, weight, residual)
    if group is not None and (group < 16 or group & (group - 1)):
        _refuse("group must be a power of two of 16 or more")
    groups = 1 if group is None else builtins.max(1, -(-cols // group))
    at = _ordinal(m, r, weight)
    q = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device)
    scales = torch.empty((*x.shape[:-1], groups), dtype=torch.float32, device=x.device)
    s = None if r is None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    check(N.lib.heph_rms_norm_fp8(at, code, m.data_ptr(), m.stride(0), _ptr(r), 0 if r is None else r.stride(0),
                                  _ptr(weight), wcode, eps, m.shape[0], cols, group or 0, q.data_ptr(),
                                  scales.data_ptr(), _ptr(s), _raw_stream(at)))
    return (q, scales) if s is None else (q, scales, s)


def rms_norm_backward(dy, s, weight=None, eps=1e-6, *, dsum=None):
    """[EXT] Gradients of rms_norm at s (its x, or the sum that it returned).

    dsum: the gradient that reaches s by other ways (the residual stream), added.  Returns
    (ds, dweight): ds in s's type, the gradient of x and of the residual alike; dweight in the
    weight's type, summed over all rows in a fixed order (None without a weight)."""
    m, cols, g, code, wcode = _norm_operands(s, weight, dy)
    d = None if dsum is None else _rows("dsum", dsum, s.shape, s.dtype)
    at = _ordinal(m, g, d, weight)
    ds = torch.empty(s.shape, dtype=s.dtype, device=s.device)
    dw = work = None
    size = 0
    if weight is not None:
        need = ctypes.c_uint64()
        check(N.lib.heph_rms_norm_backward_workspace(at, m.shape[0], cols, ctypes.byref(need)))
        size = need.value
        work = torch.empty(size, dtype=torch.uint8, device=s.device)
        dw = torch.empty(cols, dtype=weight.dtype, device=s.device)
    check(N.lib.heph_rms_norm_backward(at, code, g.data_ptr(), g.stride(0), m.data_ptr(), m.stride(0), _ptr(d),
                                       0 if d is None else d.stride(0), _ptr(weight), wcode, eps, m.shape[0], cols,
                                       ds.data_ptr(), _ptr(dw), _ptr(work), size, _raw_stream(at)))
    return ds, dw


def route_experts(logits, k, *, score="softmax", bias=None, groups=1, groups_kept=1, group_top=2, renormalize=True,
                  scale=1.0):
    """[EXT] The k experts of every row of `logits` [..., experts] and their weights.

    Scores are the logits' softmax or sigmoid; score + bias (f32 [experts]) chooses, the score
    weighs.  With groups > 1 a group of adjacent experts is worth the sum of its group_top (1 or 2)
    best choices, and only the best groups_kept groups stay.  Experts come in falling order, the
    lowest index first among equals.  renormalize divides by the sum of the chosen scores.  Returns
    (weights f32 [..., k], experts i32 [..., k]); an expert whose logit is -inf or NaN is not
    chosen, and where none is left the expert is -1 with weight 0."""
    m = _rows("logits", logits)
    rows, experts = m.shape
    if score not in _ROUTE_SCORES:
        _refuse(f"unknown routing score {score!r}")
    if bias is not None:
        _vector("bias", bias, experts, (torch.float32,))
    if not 1 <= k <= builtins.min(32, experts) or not 1 <= experts <= 1024:
        _refuse(f"route_experts chooses 1 to 32 of up to 1024 experts, not {k} of {experts}")
    at = _ordinal(m, bias)
    shape = (rows, k) if logits.dim() == 2 else (*logits.shape[:-1], k)
    weights = torch.empty(shape, dtype=torch.float32, device=m.device)
    picks = torch.empty(shape, dtype=torch.int32, device=m.device)
    check(N.lib.heph_route_experts(at, _ROW_DTYPES[m.dtype], m.data_ptr(), m.stride(0), _ptr(bias), rows, experts, k,
                                   _ROUTE_SCORES[score], groups, groups_kept, group_top, bool(renormalize), scale,
                                   weights.data_ptr(), picks.data_ptr(), _raw_stream(at)))
    return weights, picks


def route_experts_backward(dweights, logits, experts, *, score="softmax", renormalize=True, scale=1.0):
    """[EXT] Gradient of route_experts' weights by its logits, for the experts that it chose.

    dweights f32 [..., k], experts i32 [..., k] as returned.  Returns dlogits like logits (the bias
    only chooses, so it has no gradient)."""
    m = _rows("logits", logits)
    if score not in _ROUTE_SCORES:
        _refuse(f"unknown routing score {score!r}")
    if experts.dim() != logits.dim():
        _refuse("experts must have the logits' leading dimensions")
    shape = (*logits.shape[:-1], experts.shape[-1])
    g = _rows("dweights", dweights, shape, torch.float32)
    p = _rows("experts", experts, shape, torch.int32)
    at = _ordinal(m, g, p)
    dlogits = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    check(N.lib.heph_route_experts_backward(at, _ROW_DTYPES[m.dtype], g.data_ptr(), g.stride(0), m.data_ptr(),
                                            m.stride(0), p.data_ptr(), p.stride(0), m.shape[0], m.shape[1], p.shape[1],
                                            _ROUTE_SCORES[score], bool(renormalize), scale, dlogits.data_ptr(),
                                            _raw_stream(at)))
    return dlogits


def expert_order(experts, num_experts):
    """[EXT] The routed pairs of `experts` (i32, as route_experts returns it) in the order of experts.

    Returns (offsets i32 [num_experts + 1], order i32 [pairs], slot like experts): the pairs of expert
    e are order[offsets[e]:offsets[e + 1]], as places in the flattened `experts`, in rising order; slot is
    the inverse.  A pair whose expert is outside [0, num_experts) has slot -1, and order is -1 past
    the last pair."""
    if experts.dtype != torch.int32:
        _refuse(f"experts must be torch.int32, not {experts.dtype}")
    if not experts.is_contiguous():
        _refuse("experts must be contiguous")
    if not 1 <= num_experts <= 1024:
        _refuse(f"expert_order takes 1 to 1024 experts, not {num_experts}")
    at = _ordinal(experts)
    count = experts.numel()
    offsets = torch.empty(num_experts + 1, dtype=torch.int32, device=experts.device)
    order = torch.empty(count, dtype=torch.int32, device=experts.device)
    slot = torch.empty(experts.shape, dtype=torch.int32, device=experts.device)
    check(N.lib.heph_expert_order(at, experts.data_ptr(), count, num_experts, offsets.data_ptr(), order.data_ptr(),
                                  slot.data_ptr(), _raw_stream(at)))
    return offsets, order, slot


def _setting(name: str, value, rows: int, dtype):
    """(tensor or None, value) of a setting that is one number or one per row."""
    if isinstance(value, torch.Tensor):
        return _vector(name, value, rows, (dtype,)), 0
    return None, value


def sample_tokens(logits, uniform, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """[EXT] A token from every row of `logits` [rows, vocabulary], by the numbers `uniform` (f32 [rows], in [0, 1)).

    Weights are exp((l - max) / temperature).  In falling order of the logits (the lowest index first
    among equals) top_k keeps the first k (0: off), top_p of those the ones before which lies less
    than top_p of their mass (1: off), min_p of those the ones of at least min_p of the largest weight
    (0: off).  The token is the first index whose running sum of kept weights exceeds uniform times
    their whole; temperature 0 takes the largest.  Each setting is a number or a tensor of one per
    row (f32; top_k i32), where values outside its range turn it off (a temperature: take the
    largest).  The answer for a row is the same in any batch.  Returns (tokens i64 [rows], probs f32
    [rows]), the probability among the kept ones; a row of nothing but -inf and NaN has token -1."""
    m = _rows("logits", logits)
    if logits.dim() != 2 or not m.shape[1]:
        _refuse("logits must be [rows, vocabulary]")
    rows, vocab = m.shape
    _vector("uniform", uniform, rows, (torch.float32,))
    t, t_all = _setting("temperature", temperature, rows, torch.float32)
    k, k_all = _setting("top_k", top_k, rows, torch.int32)
    p, p_all = _setting("top_p", top_p, rows, torch.float32)
    least, least_all = _setting("min_p", min_p, rows, torch.float32)
    at = _ordinal(m, uniform, t, k, p, least)
    tokens = torch.empty(rows, dtype=torch.int64, device=m.device)
    probs = torch.empty(rows, dtype=torch.float32, device=m.device)
    check(N.lib.heph_sample_tokens(at, _ROW_DTYPES[m.dtype], m.data_ptr(), m.stride(0), rows, vocab, uniform.data_ptr(),
                                   _ptr(t), t_all, _ptr(k), k_all, _ptr(p), p_all, _ptr(least), least_all,
                                   tokens.data_ptr(), probs.data_ptr(), _raw_stream(at)))
    return tokens, probs
