"""Operators for token streams -- the transformer blocks that stand between channels-last features in image and video models:
``rms_norm`` (with the residual's addition in front), ``rms_norm_quant`` (leaving in 8 bits with scales), ``rotary`` (positions
with several axes, optionally behind a norm of each head) and ``clip_gradients`` / ``clip_grad_norm_``.  The reference has no
counterpart to any of them.

The kernels are those of include/gnnhwc_tokens.h in libgnnhwc_hip.so.  Ordinary eager calls run in native code
(csrc/gn_tokens_torch.cpp); what that declines -- tracing, subclasses, tensors in other layouts, and every error -- comes
here, through the ``gnop::`` operators, which carry meta kernels and autograd formulas (``clip_gradients``, which has no derivative
and works on lists, has none).
"""
import ctypes
import math

import torch
import torch.nn as nn

from . import _cabi, _native
from .custom_gn import _check_device, _current_stream_ptr, _dtype_code, _DTYPE_CODE, _on_device, _op_lib, _workspace

_POSITION_TYPE = {torch.int32: 0, torch.int64: 1, torch.float32: 2}
_QUANT_CODE = {torch.float8_e4m3fn: _cabi.F8E4M3, torch.int8: _cabi.I8}
_HALF = (torch.float16, torch.bfloat16)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _check_like(t, x, name, shape=None):
    """t has x's device and dtype, and the shape (x's unless given)."""
    _check_device(t, name)
    shape = x.shape if shape is None else shape
    if t.device != x.device or t.dtype != x.dtype or tuple(t.shape) != tuple(shape):
        raise RuntimeError("%s must be %s of shape %s on %s, got %s of shape %s on %s"
                           % (name, x.dtype, tuple(shape), x.device, t.dtype, tuple(t.shape), t.device))


def _check_weight(w, x, n, name="weight"):
    _check_device(w, name)
    if w.device != x.device or w.numel() != n:
        raise RuntimeError("%s must have %d elements on %s" % (name, n, x.device))
    if w.dtype != x.dtype and not (x.dtype in _HALF and w.dtype == torch.float32):
        raise RuntimeError("%s must be %s%s, got %s" % (name, x.dtype, " or torch.float32" if x.dtype in _HALF else "", w.dtype))
    return w.contiguous()


def _rows(t):
    """(..., C) -> (rows, C) with contiguous channels and one stride from row to row; a view where that is one."""
    if t.shape[-1] != 1 and t.stride(-1) != 1:
        t = t.contiguous()
    return t.reshape(-1, t.shape[-1])


def _stream_args(x):
    return _current_stream_ptr(x.device)


# ---- root-mean-square norm -------------------------------------------------------------------------------------------
def _check_norm(x, residual, weight, opname):
    _check_device(x, "x")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise RuntimeError("%s expects x of shape (..., C), got %s" % (opname, tuple(x.shape)))
    dt = _dtype_code(x, "x")
    if residual is not None:
        _check_like(residual, x, "residual")
    C = x.shape[-1]
    w = None if weight is None else _check_weight(weight, x, C)
    return dt, dt if w is None else _DTYPE_CODE[w.dtype], w


def _rms_norm(x, residual, weight, eps, return_sum):
    """gnop::rms_norm.  Returns (y, s); s has no elements unless there is a residual and return_sum."""
    dt, pdt, w = _check_norm(x, residual, weight, "gnop::rms_norm")
    C = x.shape[-1]
    xr, rr = _rows(x), None if residual is None else _rows(residual)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    s = torch.empty(x.shape if return_sum and residual is not None else (0,), dtype=x.dtype, device=x.device)
    with _on_device(x.device):
        rc = _cabi.lib.gnnhwc_rms_fwd(xr.data_ptr(), _ptr(rr), _ptr(w), s.data_ptr() if s.numel() else None, y.data_ptr(), xr.shape[0], C,
                                      xr.stride(0), 0 if rr is None else rr.stride(0), float(eps), dt, pdt, _stream_args(x))
    _cabi.check(rc, "gnop::rms_norm")
    return y, s


def _rms_norm_bwd(dy, ds, s, weight, eps):
    """gnop::rms_norm_bwd.  Returns (dx, dweight); dweight has no elements without a weight."""
    dt, pdt, w = _check_norm(s, None, weight, "gnop::rms_norm_bwd")
    _check_like(dy, s, "dy")
    if ds is not None:
        _check_like(ds, s, "ds")
    C = s.shape[-1]
    sr, dyr, dsr = _rows(s), _rows(dy), None if ds is None else _rows(ds)
    dx = torch.empty(s.shape, dtype=s.dtype, device=s.device)
    dw = torch.empty((C,) if w is not None else (0,), dtype=s.dtype if w is None else w.dtype, device=s.device)
    lib = _cabi.lib
    with _on_device(s.device):
        nbytes = lib.gnnhwc_rms_bwd_workspace_bytes(sr.shape[0], C, dt)
        if nbytes == 0:
            raise RuntimeError("gnop::rms_norm_bwd: " + _cabi.last_error())
        stream = _stream_args(s)
        ws = _workspace(nbytes, s.device)
        rc = lib.gnnhwc_rms_bwd(dyr.data_ptr(), _ptr(dsr), sr.data_ptr(), _ptr(w), dx.data_ptr(), dw.data_ptr() if w is not None else None,
                                sr.shape[0], C, dyr.stride(0), 0 if dsr is None else dsr.stride(0), sr.stride(0), float(eps), dt, pdt,
                                ws.data_ptr(), ws.numel(), stream)
    _cabi.check(rc, "gnop::rms_norm_bwd")
    return dx, dw


def _scale_shape(x, block):
    C = x.shape[-1]
    return (*x.shape[:-1], 1 if block == 0 or block >= C else -(-C // block))


def _rms_norm_quant(x, residual, weight, eps, block, out_dtype, return_sum):
    """gnop::rms_norm_quant.  Returns (q, scales, s); block 0: one scale per row."""
    dt, pdt, w = _check_norm(x, residual, weight, "gnop::rms_norm_quant")
    if out_dtype not in _QUANT_CODE:
        raise RuntimeError("out_dtype must be torch.float8_e4m3fn or torch.int8, got %s" % (out_dtype,))
    C = x.shape[-1]
    xr, rr = _rows(x), None if residual is None else _rows(residual)
    q = torch.empty(x.shape, dtype=out_dtype, device=x.device)
    scales = torch.empty(_scale_shape(x, block), dtype=torch.float32, device=x.device)
    s = torch.empty(x.shape if return_sum and residual is not None else (0,), dtype=x.dtype, device=x.device)
    with _on_device(x.device):
        rc = _cabi.lib.gnnhwc_rms_fwd_quant(xr.data_ptr(), _ptr(rr), _ptr(w), s.data_ptr() if s.numel() else None, q.data_ptr(),
                                            scales.data_ptr(), xr.shape[0], C, xr.stride(0), 0 if rr is None else rr.stride(0), block,
                                            float(eps), dt, pdt, _QUANT_CODE[out_dtype], _stream_args(x))
    _cabi.check(rc, "gnop::rms_norm_quant")
    return q, scales, s


_op_lib.define("rms_norm(Tensor x, Tensor? residual, Tensor? weight, float eps, bool return_sum) -> (Tensor, Tensor)")
_op_lib.define("rms_norm_bwd(Tensor dy, Tensor? ds, Tensor s, Tensor? weight, float eps) -> (Tensor, Tensor)")
_op_lib.define("rms_norm_quant(Tensor x, Tensor? residual, Tensor? weight, float eps, int block, ScalarType out_dtype, bool return_sum) "
               "-> (Tensor, Tensor, Tensor)")
_op_lib.impl("rms_norm", _rms_norm, "CompositeExplicitAutograd")
_op_lib.impl("rms_norm_bwd", _rms_norm_bwd, "CompositeExplicitAutograd")
_op_lib.impl("rms_norm_quant", _rms_norm_quant, "CompositeExplicitAutograd")


def _rms_norm_meta(x, residual, weight, eps, return_sum):
    return (torch.empty(x.shape, dtype=x.dtype, device=x.device),
            torch.empty(x.shape if return_sum and residual is not None else (0,), dtype=x.dtype, device=x.device))


def _rms_norm_bwd_meta(dy, ds, s, weight, eps):
    return (torch.empty(s.shape, dtype=s.dtype, device=s.device),
            torch.empty((s.shape[-1],) if weight is not None else (0,), dtype=s.dtype if weight is None else weight.dtype, device=s.device))


def _rms_norm_quant_meta(x, residual, weight, eps, block, out_dtype, return_sum):
    return (torch.empty(x.shape, dtype=out_dtype, device=x.device), torch.empty(_scale_shape(x, block), dtype=torch.float32, device=x.device),
            torch.empty(x.shape if return_sum and residual is not None else (0,), dtype=x.dtype, device=x.device))


_op_lib.impl("rms_norm", _rms_norm_meta, "Meta")
_op_lib.impl("rms_norm_bwd", _rms_norm_bwd_meta, "Meta")
_op_lib.impl("rms_norm_quant", _rms_norm_quant_meta, "Meta")


def _rms_norm_setup_context(ctx, inputs, output):
    x, residual, weight, ctx.eps, return_sum = inputs
    ctx.has_residual = residual is not None
    ctx.have_sum = ctx.has_residual and return_sum
    # the backward differentiates at the sum: kept if it was written, else rebuilt from the inputs
    ctx.save_for_backward(output[1] if ctx.have_sum else x, residual if ctx.has_residual and not ctx.have_sum else None, weight)
    ctx.weight_shape = None if weight is None else weight.shape
    ctx.set_materialize_grads(False)


def _rms_norm_backward(ctx, dy, ds):
    s, residual, weight = ctx.saved_tensors
    if residual is not None:
        s = (s.double() + residual.double() if s.dtype == torch.float64 else s.float() + residual.float()).to(s.dtype)
    if not ctx.have_sum:
        ds = None
    if dy is None:  # only the sum was used
        return ds, ds if ctx.has_residual else None, None, None, None
    dx, dw = torch.ops.gnop.rms_norm_bwd(dy, ds, s, weight, ctx.eps)
    return dx, dx if ctx.has_residual else None, dw.view(ctx.weight_shape) if weight is not None else None, None, None


torch.library.register_autograd("gnop::rms_norm", _rms_norm_backward, setup_context=_rms_norm_setup_context, lib=_op_lib)


def _wide(t):
    """t in the type that the kernels compute in."""
    return t if t.dtype == torch.float64 else t.float()


def _norm_second(d, t, weight, eps, a, b):
    """Gradients with respect to d, t and weight of <a, dt> + <b, dw>, where dt and dw are the norm's own gradients,
      dt = r (g - h mean(g h)),  dw = sum d h,  g = d w, h = t r;
    a or b may be None.  The map from g to dt is symmetric, which gives the parts of d and weight; with dr / dt = -r^2 h / C,
      -r^2 (h (mean(a g) - 3 mean(a h) mean(g h)) + a mean(g h) + g mean(a h))
    is that of t.  Elementary operations on _wide tensors: differentiable in their turn."""
    def mean(v):
        return v.mean(-1, keepdim=True)

    r = (mean(t * t) + eps).rsqrt()
    h = t * r
    of_d = of_t = of_w = None
    if a is not None:
        g = d if weight is None else d * weight
        ah, gh = mean(a * h), mean(g * h)
        back = r * (a - h * ah)
        of_d = back if weight is None else back * weight
        of_t = -r * r * (h * (mean(a * g) - 3 * ah * gh) + a * gh + g * ah)
        of_w = None if weight is None else (back * d).reshape(-1, t.shape[-1]).sum(0)
    if b is not None:
        e = b * d
        of_d = b * h if of_d is None else of_d + b * h
        back = r * (e - h * mean(e * h))
        of_t = back if of_t is None else of_t + back
    return of_d, of_t, of_w


def _second(d, t, weight, eps, a, b):
    """_norm_second of tensors in any type, each result in its tensor's type and shape; None where there is none."""
    if a is None and b is None:
        return None, None, None
    w = None if weight is None else _wide(weight).reshape(-1)
    grads = _norm_second(_wide(d), _wide(t), w, eps, None if a is None else _wide(a), None if b is None else _wide(b))
    return tuple(None if g is None else g.view(like.shape).to(like.dtype) for g, like in zip(grads, (d, t, weight)))


def _rms_norm_bwd_setup_context(ctx, inputs, output):
    dy, ds, s, weight, ctx.eps = inputs
    ctx.has_ds = ds is not None
    ctx.save_for_backward(dy, s, weight)
    ctx.set_materialize_grads(False)
    if weight is None:
        ctx.mark_non_differentiable(output[1])


def _rms_norm_bwd_backward(ctx, a, b):
    dy, s, weight = ctx.saved_tensors
    of_dy, of_s, of_weight = _second(dy, s, weight, ctx.eps, a, None if weight is None else b)
    return of_dy, a if ctx.has_ds else None, of_s, of_weight, None


torch.library.register_autograd("gnop::rms_norm_bwd", _rms_norm_bwd_backward, setup_context=_rms_norm_bwd_setup_context, lib=_op_lib)


def _needs_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def rms_norm(x, weight=None, eps=1e-6, residual=None, return_sum=False, channel_dim=-1):
    """s / sqrt(mean(s^2) + eps) * weight over the channels, s = x + residual.

    x: (..., C) -- or any layout with the channels at `channel_dim`, e.g. 1 for (N, C, H, W) in channels-last memory, which is
    taken as it is; float32, float64, float16 or bfloat16, C up to 16384 (float64: 8192).  weight: (C,) in x's dtype, or float32
    beside half-precision data, or None.  residual: a tensor like x; the sum is rounded to x's dtype once, as an addition in
    front would, and is what is normalised.  With return_sum=True the call returns (y, s), so that s is the next residual
    (without a residual, s is x).  Means and products are in float32 (float64).  Differentiable in x, residual and weight, as
    often as need be (from the second derivative on in elementary operations); the gradients of s reach x and residual too."""
    if channel_dim != -1 and channel_dim != x.dim() - 1:
        last = [None if t is None else t.movedim(channel_dim, -1) for t in (x, residual)]
        out = rms_norm(last[0], weight, eps, last[1], return_sum)
        return tuple(t.movedim(-1, channel_dim) for t in out) if return_sum else out.movedim(-1, channel_dim)
    if not torch.compiler.is_compiling():
        out = _native.rms_norm(x, weight, eps, residual, return_sum)
        if out is not NotImplemented:
            return out
    want = residual is not None and (return_sum or _needs_grad(x, residual, weight))
    y, s = torch.ops.gnop.rms_norm(x, residual, weight, eps, want)
    if not return_sum:
        return y
    return y, x if residual is None else s


def rms_norm_quant(x, weight=None, eps=1e-6, residual=None, return_sum=False, out_dtype=torch.float8_e4m3fn, block=None):
    """rms_norm with the result in 8 bits for an 8-bit product: (q, scales), or (q, scales, s) with return_sum=True, such that
    q * scales is the norm.  x: (..., C) in float32, float16 or bfloat16.

    scale = max(max |y| / most, 2^-126) per row (block=None; scales are (..., 1)) or per `block` consecutive channels (a power of
    two from 16 to 256; scales are (..., ceil(C / block))), most = 448 for torch.float8_e4m3fn and 127 for torch.int8;
    q = y / scale, rounded to nearest even from float32.  For serving: it has no derivative."""
    if not torch.compiler.is_compiling():
        out = _native.rms_norm_quant(x, weight, eps, residual, return_sum, out_dtype, block)
        if out is not NotImplemented:
            return out
    if _needs_grad(x, residual, weight):
        raise RuntimeError("rms_norm_quant has no derivative: call it under torch.no_grad()")
    if block is not None and block < 1:
        raise RuntimeError("block must be None or positive")
    q, scales, s = torch.ops.gnop.rms_norm_quant(x, residual, weight, eps, block or 0, out_dtype, return_sum)
    if residual is None:
        s = x
    return (q, scales, s) if return_sum else (q, scales)


class RMSNorm(nn.RMSNorm):
    """Module of rms_norm over `num_channels` channels at `channel_dim` (1 for channels-last images (N, C, *spatial)); its
    state_dict is torch.nn.RMSNorm's.  forward(x) -> y, forward(x, residual) -> (y, x + residual)."""

    def __init__(self, num_channels, eps=1e-6, channel_dim=-1, **kwargs):
        super().__init__(num_channels, eps=eps, **kwargs)
        self.channel_dim = channel_dim

    def forward(self, x, residual=None):
        return rms_norm(x, self.weight, self.eps, residual, residual is not None, self.channel_dim)

    def extra_repr(self):
        return super().extra_repr() + (", channel_dim=%d" % self.channel_dim if self.channel_dim != -1 else "")


# ---- rotary positions ------------------------------------------------------------------------------------------------
def rotary_frequencies(sections, theta=10000.0, ladder="axis", device=None):
    """Frequencies of the pairs of a head whose sections of pairs turn by the axes' positions, float32 (sum(sections),).

    ladder="axis": every axis has its own, theta^(-i / n) for the i-th of its n pairs (images, video);
    ladder="head": they run through the whole head, theta^(-j / P), and an axis takes its stretch of them."""
    if ladder not in ("axis", "head"):
        raise ValueError("ladder must be 'axis' or 'head'")
    P, parts, at = sum(sections), [], 0
    for n in sections:
        j = torch.arange(n, dtype=torch.float64)
        parts.append(theta ** (-j / n) if ladder == "axis" else theta ** (-(j + at) / P))
        at += n
    return torch.cat(parts).float().to(device)


def _check_rotary(q, k, positions, frequencies, sections, q_weight, k_weight, opname):
    """Checks that need no memory; returns (B, L, A, positions as (B or 1, L, A))."""
    _check_device(q, "q")
    if q.dim() != 4:
        raise RuntimeError("%s expects q of shape (B, L, heads, head_dim), got %s" % (opname, tuple(q.shape)))
    B, L, H, D = q.shape
    _dtype_code(q, "q")
    if k is not None:
        _check_like(k, q, "k", (B, L, k.shape[2] if k.dim() == 4 else 1, D))
    _check_device(positions, "positions")
    _check_device(frequencies, "frequencies")
    if positions.device != q.device or frequencies.device != q.device:
        raise RuntimeError("positions and frequencies must be on %s" % q.device)
    if positions.dtype not in _POSITION_TYPE:
        raise RuntimeError("positions must be int32, int64 or float32, got %s" % positions.dtype)
    if frequencies.dtype != torch.float32 or frequencies.dim() != 1 or frequencies.numel() != sum(sections):
        raise RuntimeError("frequencies must be float32 with one value for each of the sections' %d pairs" % sum(sections))
    A = len(sections)
    if not 1 <= A <= 4 or min(sections) < 0:
        raise RuntimeError("sections must be 1 to 4 counts of pairs")
    p = positions
    if A == 1 and (p.dim() == 1 or (p.dim() == 2 and p.shape[-1] == L)):
        p = p.unsqueeze(-1)
    if p.dim() == 2:
        p = p.unsqueeze(0)
    if p.dim() != 3 or p.shape[0] not in (1, B) or p.shape[1] != L or p.shape[2] != A:
        raise RuntimeError("positions must have shape (L, axes) or (B, L, axes) = (%d, %d, %d), got %s" % (B, L, A, tuple(positions.shape)))
    if (q_weight is None) != (k_weight is None) and k is not None:
        raise RuntimeError("q_weight and k_weight must both be given or both be None")
    if k is None and k_weight is not None:
        raise RuntimeError("k_weight without k")
    return B, L, A, p


def _heads(t):
    return t if t is None or t.stride(-1) == 1 else t.contiguous()


def _strides3(t):
    return (ctypes.c_int64 * 3)(*t.stride()[:3])


def _rotary_call(q, k, p, frequencies, sections, interleaved, q_weight, k_weight, eps, keep):
    """The argument block without tensors' pointers; `keep` collects what has to live until the call."""
    B, L, H, D = q.shape
    c = _cabi.RotaryCall()
    c.batch, c.tokens, c.heads, c.kv_heads, c.head_dim = B, L, H, 0 if k is None else k.shape[2], D
    c.axes = len(sections)
    end = 0
    for i, n in enumerate(sections):
        end += n
        c.section_end[i] = end
    c.interleaved = 1 if interleaved else 0
    if p.shape[2] != 1 and p.stride(2) != 1:
        p = p.contiguous()
    frequencies = frequencies.contiguous()
    keep += [p, frequencies]
    c.positions, c.position_type = p.data_ptr(), _POSITION_TYPE[p.dtype]
    c.position_stride[0], c.position_stride[1] = (0 if p.shape[0] == 1 else p.stride(0)), p.stride(1)
    c.frequencies = frequencies.data_ptr()
    c.eps, c.dtype, c.param_dtype = float(eps), _DTYPE_CODE[q.dtype], _DTYPE_CODE[q.dtype]
    if q_weight is not None:
        qw = _check_weight(q_weight, q, D, "q_weight")
        kw = None if k is None else _check_weight(k_weight, q, D, "k_weight")
        if kw is not None and kw.dtype != qw.dtype:
            raise RuntimeError("q_weight and k_weight must have the same dtype")
        keep += [qw, kw]
        c.q_weight, c.k_weight, c.param_dtype = qw.data_ptr(), _ptr(kw), _DTYPE_CODE[qw.dtype]
    return c


def _rotary(q, k, positions, frequencies, sections, interleaved, q_weight, k_weight, eps):
    """gnop::rotary.  Returns (q_out, k_out) contiguous; k_out has no elements without k."""
    B, L, _A, p = _check_rotary(q, k, positions, frequencies, sections, q_weight, k_weight, "gnop::rotary")
    keep = []
    c = _rotary_call(q, k, p, frequencies, sections, interleaved, q_weight, k_weight, eps, keep)
    q, k = _heads(q), _heads(k)
    qo = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    ko = torch.empty(k.shape if k is not None else (0,), dtype=q.dtype, device=q.device)
    c.q, c.q_out, c.q_stride, c.q_out_stride = q.data_ptr(), qo.data_ptr(), _strides3(q), _strides3(qo)
    if k is not None:
        c.k, c.k_out, c.k_stride, c.k_out_stride = k.data_ptr(), ko.data_ptr(), _strides3(k), _strides3(ko)
    with _on_device(q.device):
        rc = _cabi.lib.gnnhwc_rotary(ctypes.byref(c), _stream_args(q))
    _cabi.check(rc, "gnop::rotary")
    return qo, ko


def _rotary_bwd(q_grad, k_grad, q, k, positions, frequencies, sections, interleaved, q_weight, k_weight, eps):
    """gnop::rotary_bwd.  q and k are read only where there are weights.  Returns (dq, dk, dq_weight, dk_weight)."""
    _B, _L, _A, p = _check_rotary(q_grad, k_grad, positions, frequencies, sections, q_weight, k_weight, "gnop::rotary_bwd")
    keep = []
    c = _rotary_call(q_grad, k_grad, p, frequencies, sections, interleaved, q_weight, k_weight, eps, keep)
    norm = q_weight is not None
    if norm:
        if q is None or (k is None) != (k_grad is None):
            raise RuntimeError("gnop::rotary_bwd behind a norm needs q and k")
        _check_like(q, q_grad, "q")
        q = _heads(q)
        c.q, c.q_stride = q.data_ptr(), _strides3(q)
        if k is not None:
            _check_like(k, k_grad, "k")
            k = _heads(k)
            c.k, c.k_stride = k.data_ptr(), _strides3(k)
    q_grad, k_grad = _heads(q_grad), _heads(k_grad)
    dev, dtype = q_grad.device, q_grad.dtype
    D = q_grad.shape[-1]
    dq = torch.empty(q_grad.shape, dtype=dtype, device=dev)
    dk = torch.empty(k_grad.shape if k_grad is not None else (0,), dtype=dtype, device=dev)
    dqw = torch.empty((D if norm else 0,), dtype=q_weight.dtype if norm else dtype, device=dev)
    dkw = torch.empty((D if norm and k_grad is not None else 0,), dtype=dqw.dtype, device=dev)
    c.q_grad, c.q_out, c.q_grad_stride, c.q_out_stride = q_grad.data_ptr(), dq.data_ptr(), _strides3(q_grad), _strides3(dq)
    if k_grad is not None:
        c.k_grad, c.k_out, c.k_grad_stride, c.k_out_stride = k_grad.data_ptr(), dk.data_ptr(), _strides3(k_grad), _strides3(dk)
    lib = _cabi.lib
    with _on_device(dev):
        stream = _stream_args(q_grad)
        ws_ptr, ws_bytes = None, 0
        if norm:
            c.q_dweight, c.k_dweight = dqw.data_ptr(), dkw.data_ptr() if dkw.numel() else None
            nbytes = lib.gnnhwc_rotary_bwd_workspace_bytes(ctypes.byref(c))
            if nbytes == 0:
                raise RuntimeError("gnop::rotary_bwd: " + _cabi.last_error())
            ws = _workspace(nbytes, dev)
            ws_ptr, ws_bytes = ws.data_ptr(), ws.numel()
        rc = lib.gnnhwc_rotary_bwd(ctypes.byref(c), ws_ptr, ws_bytes, stream)
    _cabi.check(rc, "gnop::rotary_bwd")
    return dq, dk, dqw, dkw


_op_lib.define("rotary(Tensor q, Tensor? k, Tensor positions, Tensor frequencies, int[] sections, bool interleaved, Tensor? q_weight, "
               "Tensor? k_weight, float eps) -> (Tensor, Tensor)")
_op_lib.define("rotary_bwd(Tensor q_grad, Tensor? k_grad, Tensor? q, Tensor? k, Tensor positions, Tensor frequencies, int[] sections, "
               "bool interleaved, Tensor? q_weight, Tensor? k_weight, float eps) -> (Tensor, Tensor, Tensor, Tensor)")
_op_lib.impl("rotary", _rotary, "CompositeExplicitAutograd")
_op_lib.impl("rotary_bwd", _rotary_bwd, "CompositeExplicitAutograd")


def _rotary_meta(q, k, positions, frequencies, sections, interleaved, q_weight, k_weight, eps):
    return (torch.empty(q.shape, dtype=q.dtype, device=q.device), torch.empty(k.shape if k is not None else (0,), dtype=q.dtype, device=q.device))


def _rotary_bwd_meta(q_grad, k_grad, q, k, positions, frequencies, sections, interleaved, q_weight, k_weight, eps):
    D, dev, dtype = q_grad.shape[-1], q_grad.device, q_grad.dtype
    wtype = dtype if q_weight is None else q_weight.dtype
    return (torch.empty(q_grad.shape, dtype=dtype, device=dev), torch.empty(k_grad.shape if k_grad is not None else (0,), dtype=dtype, device=dev),
            torch.empty((D if q_weight is not None else 0,), dtype=wtype, device=dev),
            torch.empty((D if k_weight is not None else 0,), dtype=wtype, device=dev))


_op_lib.impl("rotary", _rotary_meta, "Meta")
_op_lib.impl("rotary_bwd", _rotary_bwd_meta, "Meta")


def _rotary_setup_context(ctx, inputs, output):
    q, k, positions, frequencies, ctx.sections, ctx.interleaved, q_weight, k_weight, ctx.eps = inputs
    norm = q_weight is not None
    ctx.has_k = k is not None
    ctx.save_for_backward(q if norm else None, k if norm else None, positions, frequencies, q_weight, k_weight)
    ctx.shapes = None if q_weight is None else (q_weight.shape, k_weight.shape if k_weight is not None else None)
    if not ctx.has_k:
        ctx.mark_non_differentiable(output[1])


def _rotary_backward(ctx, dq, dk):
    q, k, positions, frequencies, q_weight, k_weight = ctx.saved_tensors
    gq, gk, gqw, gkw = torch.ops.gnop.rotary_bwd(dq, dk if ctx.has_k else None, q, k, positions, frequencies, ctx.sections, ctx.interleaved,
                                                 q_weight, k_weight, ctx.eps)
    return (gq, gk if ctx.has_k else None, None, None, None, None, gqw.view(ctx.shapes[0]) if q_weight is not None else None,
            gkw.view(ctx.shapes[1]) if k_weight is not None else None, None)


torch.library.register_autograd("gnop::rotary", _rotary_backward, setup_context=_rotary_setup_context, lib=_op_lib)


def _rotary_bwd_setup_context(ctx, inputs, output):
    q_grad, k_grad, q, k, positions, frequencies, ctx.sections, ctx.interleaved, q_weight, k_weight, ctx.eps = inputs
    norm = q_weight is not None
    ctx.norm, ctx.has_k = norm, k_grad is not None
    # (without a norm the gradients are linear in the incoming ones, and nothing else is differentiated)
    ctx.save_for_backward(positions, frequencies, *((q_grad, k_grad, q, k, q_weight, k_weight) if norm else ()))
    ctx.set_materialize_grads(False)
    absent = [t for t, there in zip(output, (True, ctx.has_k, norm, norm and ctx.has_k)) if not there]
    ctx.mark_non_differentiable(*absent)


def _rotary_bwd_backward(ctx, *grads):
    positions, frequencies, *rest = ctx.saved_tensors
    turn = (positions, frequencies, ctx.sections, ctx.interleaved, None, None, ctx.eps)

    def side(i, there):
        """Gradients with respect to the incoming gradient, the heads and the weight of q (0) or k (1)."""
        a, b = grads[i], grads[2 + i]
        if not there or (a is None and (b is None or not ctx.norm)):
            return None, None, None
        if not ctx.norm:
            return torch.ops.gnop.rotary(a, None, *turn)[0], None, None
        g, t, w = rest[i], rest[2 + i], rest[4 + i]
        d = torch.ops.gnop.rotary_bwd(_wide(g), None, None, None, *turn)[0]  # behind the turn, in front of the norm
        of_d, of_t, of_w = _second(d, t, w, ctx.eps, a, b)
        return torch.ops.gnop.rotary(of_d, None, *turn)[0].to(g.dtype), of_t, of_w

    (gq, tq, wq), (gk, tk, wk) = side(0, True), side(1, ctx.has_k)
    return gq, gk, tq, tk, None, None, None, None, wq, wk, None


torch.library.register_autograd("gnop::rotary_bwd", _rotary_bwd_backward, setup_context=_rotary_bwd_setup_context, lib=_op_lib)


def rotary(q, k, positions, frequencies, sections=None, interleaved=False, q_weight=None, k_weight=None, eps=1e-6):
    """Rotary positions with one to four axes (time, height, width, ...) on q and k.  Returns (q', k'), or q' if k is None.

    q: (B, L, heads, D), k: (B, L, kv_heads, D) or None, with any strides as long as a head's channels are contiguous (slices of
    one packed projection are read where they are); D even, up to 256.  positions: (L, axes) or (B, L, axes), int32, int64 or
    float32, whole numbers within 32 bits and exact to 2^24 (with one axis also (L,) or (B, L)).  frequencies: float32, one for
    each turning pair, see rotary_frequencies; sections: how many of them belong to each axis, in order (None: all to one axis).
    Pair j of a head is its channels (2 j, 2 j + 1) if `interleaved`, else (j, j + P), P = sum(sections); it is turned by
    positions[axis] * frequencies[j].  Channels behind the 2 P first stay as they are.

    With q_weight / k_weight, (D,) in q's dtype or float32 beside half precision, every head is first normalised over its D
    channels, t / sqrt(mean(t^2) + eps) * weight, in the same pass.  Everything in between is float32 (float64).
    Differentiable in q, k and the weights, as often as need be (behind a norm from the second derivative on in elementary
    operations)."""
    if not torch.compiler.is_compiling():
        out = _native.rotary(q, k, positions, frequencies, sections, interleaved, q_weight, k_weight, eps)
        if out is not NotImplemented:
            return out
    sections = (frequencies.numel(),) if sections is None else tuple(int(n) for n in sections)
    qo, ko = torch.ops.gnop.rotary(q, k, positions, frequencies, sections, bool(interleaved), q_weight, k_weight, float(eps))
    return qo if k is None else (qo, ko)


class Rotary(nn.Module):
    """Module of `rotary` for heads of `head_dim` channels whose `sections` of pairs turn by the positions' axes; with
    qk_norm=True it owns the weights of a norm of q's and k's heads.  forward(q, k, positions) -> (q', k')."""

    def __init__(self, head_dim, sections, theta=10000.0, ladder="axis", interleaved=False, qk_norm=False, eps=1e-6, device=None, dtype=None):
        super().__init__()
        self.head_dim, self.sections, self.interleaved, self.eps = head_dim, tuple(int(n) for n in sections), interleaved, eps
        if 2 * sum(self.sections) > head_dim:
            raise ValueError("sections hold %d pairs, a head of %d channels has %d" % (sum(self.sections), head_dim, head_dim // 2))
        self.register_buffer("frequencies", rotary_frequencies(self.sections, theta, ladder, device), persistent=False)
        for name in ("q_weight", "k_weight"):
            self.register_parameter(name, nn.Parameter(torch.ones(head_dim, device=device, dtype=dtype)) if qk_norm else None)

    def _apply(self, fn, recurse=True):
        # module.half() / .bfloat16() leave the angles' frequencies in float32
        kept = self.frequencies
        super()._apply(fn, recurse)
        if self.frequencies.dtype != torch.float32:
            self.frequencies = kept.to(self.frequencies.device)
        return self

    def forward(self, q, k, positions):
        return rotary(q, k, positions, self.frequencies, self.sections, self.interleaved, self.q_weight, self.k_weight, self.eps)

    def extra_repr(self):
        return "%d, sections=%s, interleaved=%s, qk_norm=%s" % (self.head_dim, self.sections, self.interleaved, self.q_weight is not None)


# ---- gradient clipping -----------------------------------------------------------------------------------------------
def _dense(t):
    """t's elements fill one stretch of memory (in whatever order of dimensions)."""
    if t.is_contiguous():
        return True
    expect = 1
    for n, s in sorted(((n, s) for n, s in zip(t.shape, t.stride()) if n != 1), key=lambda d: d[1]):
        if s != expect:
            return False
        expect *= n
    return True


def clip_gradients(grads, max_norm, out=None, grad_scale=1.0, eps=1e-6):
    """The Euclidean norm over all tensors of `grads`, and their clipping to `max_norm`; returns the norm as a tensor on the
    device (nothing waits for it).

      total = |grad_scale| * sqrt(sum of squares),   result = grad * (grad_scale * min(1, max_norm / (total + eps)))

    grads: tensors on one device, any floating types and dense layouts (channels-last included), mixed.  out=None: in place;
    else tensors like the gradients, in any floating types, that receive the results (e.g. float32 ones of half-precision
    gradients).  grad_scale: the reciprocal of a loss scale.  max_norm=math.inf computes the norm only (unless out or
    grad_scale ask for more).  As the formula has it, a norm that is NaN gives NaN throughout, and an infinite one zeros for what
    is finite and NaN for what is not.  Squares are summed in float64, in a fixed order; the norm is float32 (float64 if all
    gradients are).  An ordinary function on lists, not an operator of torch.library: it is called outside compiled graphs."""
    grads = list(grads)
    outs = None if out is None else list(out)
    if outs is not None and len(outs) != len(grads):
        raise RuntimeError("out must have as many tensors as grads")
    if not grads:
        return torch.zeros(())
    result = _native.clip_gradients(grads, float(max_norm), outs, float(grad_scale), float(eps))
    if result is not NotImplemented:
        return result
    with torch.no_grad():
        return _clip_general(grads, outs, max_norm, grad_scale, eps)


def _check_written(t, name):
    if any(n > 1 and s == 0 for n, s in zip(t.shape, t.stride())):  # an expanded tensor
        raise RuntimeError("%s cannot be written: its elements share memory" % name)


def _clip_general(grads, outs, max_norm, grad_scale, eps):
    dev = grads[0].device
    keep, back = [], []
    changes = outs is not None or grad_scale != 1.0 or max_norm < math.inf
    for i, g in enumerate(grads):
        _check_device(g, "gradient %d" % i)
        _dtype_code(g, "gradient %d" % i)
        if g.layout != torch.strided or g.device != dev:
            raise RuntimeError("gradient %d must be a dense tensor on %s" % (i, dev))
        if outs is None:
            if changes:
                _check_written(g, "gradient %d" % i)
            if not _dense(g) or g.is_neg():  # a slice with gaps, or a view that only stands for negated memory: through a copy
                c = g.resolve_neg().contiguous()
                if changes:
                    back.append((g, c))
                g = c
            keep.append((g, g))
            continue
        o = outs[i]
        _check_device(o, "out %d" % i)
        _dtype_code(o, "out %d" % i)
        if o.shape != g.shape or o.device != dev or o.layout != torch.strided:
            raise RuntimeError("out %d must have the gradient's shape %s on %s" % (i, tuple(g.shape), dev))
        _check_written(o, "out %d" % i)
        g = g.resolve_neg()
        if not (_dense(g) and _dense(o) and not o.is_neg() and (g.stride() == o.stride() or g.is_contiguous() and o.is_contiguous())):
            g = g.contiguous()
            if not o.is_contiguous() or o.is_neg():
                c = torch.empty(o.shape, dtype=o.dtype, device=dev)
                back.append((o, c))
                o = c
        keep.append((g, o))
    n = len(keep)
    total = torch.empty((), dtype=torch.float64 if all(g.dtype == torch.float64 for g, _ in keep) else torch.float32, device=dev)
    ins = (ctypes.c_void_p * n)(*[g.data_ptr() for g, _ in keep])
    sizes = (ctypes.c_int64 * n)(*[g.numel() for g, _ in keep])
    types = (ctypes.c_int * n)(*[_DTYPE_CODE[g.dtype] for g, _ in keep])
    to = None if outs is None else (ctypes.c_void_p * n)(*[o.data_ptr() for _, o in keep])
    to_types = None if outs is None else (ctypes.c_int * n)(*[_DTYPE_CODE[o.dtype] for _, o in keep])
    lib = _cabi.lib
    with _on_device(dev):
        stream = _current_stream_ptr(dev)
        ws = _workspace(lib.gnnhwc_clip_workspace_bytes(n), dev)
        rc = lib.gnnhwc_clip(ins, to, sizes, types, to_types, n, float(max_norm), float(eps), float(grad_scale), total.data_ptr(),
                             _DTYPE_CODE[total.dtype], ws.data_ptr(), ws.numel(), stream)
    _cabi.check(rc, "clip_gradients")
    for t, c in back:
        t.copy_(c)
    if changes:
        torch.autograd.graph.increment_version([t for t in (grads if outs is None else outs) if not t.is_inference()])
    return total


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, *, grad_scale=1.0, eps=1e-6):
    """clip_gradients in place over the gradients of `parameters` (a parameter that is listed twice counts once).  The first
    three arguments are those of torch.nn.utils.clip_grad_norm_; the Euclidean norm is the only norm_type."""
    if norm_type != 2:
        raise RuntimeError("clip_grad_norm_: norm_type must be 2, got %s" % (norm_type,))
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    unique = {id(p): p for p in parameters}.values()
    return clip_gradients([p.grad for p in unique if p.grad is not None], math.inf if max_norm is None else max_norm, None, grad_scale, eps)
