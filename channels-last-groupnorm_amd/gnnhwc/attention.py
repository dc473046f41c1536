"""Attention of token streams: ``window_attention``, in which a token sees a window around it and a few first tokens (registers,
sinks) that stay visible, and ``window_attention_cached``, the same for the newest tokens of each request against its cache.  The
reference has no counterpart to either.

The kernels are those of include/gnnhwc_tokens.h in libgnnhwc_hip.so.  Ordinary eager calls run in native code
(csrc/gn_tokens_torch.cpp); what that declines -- tracing, subclasses, tensors in other layouts, and every error -- comes here,
through the ``gnop::`` operators, which carry meta kernels and the autograd formula.
"""
import ctypes
import math

import torch
import torch.nn.functional as F

from . import _cabi, _native
from .custom_gn import _check_device, _current_stream_ptr, _DTYPE_CODE, _on_device, _op_lib, _workspace

_TYPES = (torch.float32, torch.float16, torch.bfloat16)


def _check_attention(q, k, v, lengths, window, sinks, at_end, opname):
    for t, name in ((q, "q"), (k, "k"), (v, "v")):
        _check_device(t, name)
        if t.dim() != 4:
            raise RuntimeError("%s expects %s of shape (B, tokens, heads, head_dim), got %s" % (opname, name, tuple(t.shape)))
        if t.dtype not in _TYPES or t.dtype != q.dtype or t.device != q.device:
            raise RuntimeError("%s takes q, k and v in float32, float16 or bfloat16, of one type and on one device; %s is %s on %s"
                               % (opname, name, t.dtype, t.device))
    B, L, H, D = q.shape
    S, K = k.shape[1], k.shape[2]
    if tuple(k.shape) != (B, S, K, D) or v.shape != k.shape:
        raise RuntimeError("%s: k and v must have shape (%d, tokens, kv_heads, %d), got %s and %s" % (opname, B, D, tuple(k.shape), tuple(v.shape)))
    if K < 1 or H < 1 or H % K:
        raise RuntimeError("%s: q's %d heads must be a multiple of k's %d" % (opname, H, K))
    most = 128 if q.dtype == torch.float32 else 256
    if not 1 <= D <= most:
        raise RuntimeError("%s: heads of %d channels: 1 to %d are supported in %s" % (opname, D, most, q.dtype))
    if not at_end and L > S:
        raise RuntimeError("%s: %d queries and %d keys: the queries are the last of the keys' tokens" % (opname, L, S))
    if window < -1 or sinks < 0:
        raise RuntimeError("%s: window and sinks must not be negative" % opname)
    if lengths is not None:
        _check_device(lengths, "lengths")
        if lengths.device != q.device or lengths.dtype not in (torch.int32, torch.int64) or tuple(lengths.shape) != (B,):
            raise RuntimeError("%s: lengths must be int32 or int64 of shape (%d,) on %s" % (opname, B, q.device))


def _aligned(t):
    """t as the kernels read it: whole 16 bytes between its rows and in front; a copy where it is laid out otherwise."""
    n = 16 // t.element_size()
    if t.numel() == 0 or (t.stride(3) == 1 and t.data_ptr() % 16 == 0 and all(s % n == 0 or m == 1 for m, s in zip(t.shape[:3], t.stride()))
                          and (t.shape[1] == 1 or t.stride(1) * t.element_size() < 2 ** 25)):
        return t
    # (a contiguous tensor may start anywhere, too)
    return torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t)


def _strides3(t):
    return (ctypes.c_int64 * 3)(*t.stride()[:3])


def _call(q, k, v, lengths, window, sinks, causal, at_end, scale, keep):
    c = _cabi.WindowCall()
    B, L, H, D = q.shape
    q, k, v = _aligned(q), _aligned(k), _aligned(v)
    keep += [q, k, v]
    c.q, c.k, c.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
    c.q_stride, c.k_stride, c.v_stride = _strides3(q), _strides3(k), _strides3(v)
    c.batch, c.tokens, c.keys, c.heads, c.kv_heads, c.head_dim = B, L, k.shape[1], H, k.shape[2], D
    c.window, c.sinks, c.causal, c.at_end = window, sinks, 1 if causal else 0, 1 if at_end else 0
    if lengths is not None:
        lengths = lengths.contiguous()
        keep.append(lengths)
        c.lengths, c.length_type = lengths.data_ptr(), 0 if lengths.dtype == torch.int32 else 1
    c.scale, c.dtype = float(scale), _DTYPE_CODE[q.dtype]
    return c


def _window_attention(q, k, v, lengths, window, sinks, causal, at_end, scale, want_lse):
    """gnop::window_attention.  Returns (out, lse, rest): what the backward reads; the last two have no elements unless it is to run
    (want_lse), rest, which is what rounding left of out, none in float32 either."""
    opname = "gnop::window_attention"
    _check_attention(q, k, v, lengths, window, sinks, at_end, opname)
    keep = []
    c = _call(q, k, v, lengths, window, sinks, causal, at_end, scale, keep)
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty((q.shape[0], q.shape[2], q.shape[1]) if want_lse else (0,), dtype=torch.float32, device=q.device)
    rest = torch.empty(_rest_shape(q, want_lse), dtype=q.dtype, device=q.device)
    c.out, c.out_stride, c.lse = out.data_ptr(), _strides3(out), lse.data_ptr() if want_lse else None
    c.out_rest = rest.data_ptr() if rest.numel() else None
    lib = _cabi.lib
    with _on_device(q.device):
        nbytes = lib.gnnhwc_window_workspace_bytes(ctypes.byref(c))
        if nbytes == 0:
            raise RuntimeError(opname + ": " + _cabi.last_error())
        ws = _workspace(nbytes, q.device)
        rc = lib.gnnhwc_window(ctypes.byref(c), ws.data_ptr(), ws.numel(), _current_stream_ptr(q.device))
    _cabi.check(rc, opname)
    return out, lse, rest


def _rest_shape(q, want_lse):
    return q.shape if want_lse and q.dtype != torch.float32 else (0,)


def _check_kept(q, lse, rest, opname):
    """What the forward left for the backward, which the kernels read by q's sizes."""
    B, L, H, _ = q.shape
    if tuple(lse.shape) != (B, H, L) or lse.dtype != torch.float32 or lse.device != q.device:
        raise RuntimeError("%s: lse must be float32 of shape %s on %s, as the forward leaves it with want_lse" % (opname, (B, H, L), q.device))
    if rest.numel() and (rest.shape != q.shape or rest.dtype != q.dtype or rest.device != q.device):
        raise RuntimeError("%s: rest must be like q, or empty" % opname)


def _window_attention_bwd(dout, q, k, v, out, lse, rest, lengths, window, sinks, causal, scale):
    """gnop::window_attention_bwd.  Returns (dq, dk, dv)."""
    opname = "gnop::window_attention_bwd"
    _check_attention(q, k, v, lengths, window, sinks, False, opname)
    for t, name in ((dout, "dout"), (out, "out")):
        _check_device(t, name)
        if t.shape != q.shape or t.dtype != q.dtype or t.device != q.device:
            raise RuntimeError("%s: %s must be like q" % (opname, name))
    _check_kept(q, lse, rest, opname)
    keep = []
    c = _call(q, k, v, lengths, window, sinks, causal, False, scale, keep)
    dout, out, lse = _aligned(dout), _aligned(out), lse.contiguous()
    rest = _aligned(rest.contiguous())
    c.out_rest = rest.data_ptr() if rest.numel() else None
    dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
    c.out, c.out_stride, c.out_grad, c.out_grad_stride, c.lse = out.data_ptr(), _strides3(out), dout.data_ptr(), _strides3(dout), lse.data_ptr()
    c.q_grad, c.q_grad_stride, c.k_grad, c.k_grad_stride = dq.data_ptr(), _strides3(dq), dk.data_ptr(), _strides3(dk)
    c.v_grad, c.v_grad_stride = dv.data_ptr(), _strides3(dv)
    lib = _cabi.lib
    with _on_device(q.device):
        nbytes = lib.gnnhwc_window_bwd_workspace_bytes(ctypes.byref(c))
        if nbytes == 0:
            raise RuntimeError(opname + ": " + _cabi.last_error())
        ws = _workspace(nbytes, q.device)
        rc = lib.gnnhwc_window_bwd(ctypes.byref(c), ws.data_ptr(), ws.numel(), _current_stream_ptr(q.device))
    _cabi.check(rc, opname)
    return dq, dk, dv


_op_lib.define("window_attention(Tensor q, Tensor k, Tensor v, Tensor? lengths, int window, int sinks, bool causal, bool at_end, float scale, "
               "bool want_lse) -> (Tensor, Tensor, Tensor)")
_op_lib.define("window_attention_bwd(Tensor dout, Tensor q, Tensor k, Tensor v, Tensor out, Tensor lse, Tensor rest, Tensor? lengths, int window, int sinks, "
               "bool causal, float scale) -> (Tensor, Tensor, Tensor)")
_op_lib.impl("window_attention", _window_attention, "CompositeExplicitAutograd")
_op_lib.impl("window_attention_bwd", _window_attention_bwd, "CompositeExplicitAutograd")


def _window_attention_meta(q, k, v, lengths, window, sinks, causal, at_end, scale, want_lse):
    return (torch.empty(q.shape, dtype=q.dtype, device=q.device),
            torch.empty((q.shape[0], q.shape[2], q.shape[1]) if want_lse else (0,), dtype=torch.float32, device=q.device),
            torch.empty(_rest_shape(q, want_lse), dtype=q.dtype, device=q.device))


def _window_attention_bwd_meta(dout, q, k, v, out, lse, rest, lengths, window, sinks, causal, scale):
    return tuple(torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))


_op_lib.impl("window_attention", _window_attention_meta, "Meta")
_op_lib.impl("window_attention_bwd", _window_attention_bwd_meta, "Meta")


def _setup_context(ctx, inputs, output):
    q, k, v, lengths, ctx.window, ctx.sinks, ctx.causal, ctx.at_end, ctx.scale, ctx.have_lse = inputs
    ctx.save_for_backward(q, k, v, *output, lengths)
    ctx.mark_non_differentiable(output[1], output[2])
    ctx.set_materialize_grads(False)


def _backward(ctx, dout, _dlse, _drest):
    if ctx.at_end or not ctx.have_lse:
        raise RuntimeError("gnop::window_attention: attention against a cache, or without lse, has no derivative")
    if dout is None:
        return (None,) * 10
    q, k, v, out, lse, rest, lengths = ctx.saved_tensors
    grads = torch.ops.gnop.window_attention_bwd(dout, q, k, v, out, lse, rest, lengths, ctx.window, ctx.sinks, ctx.causal, ctx.scale)
    return (*grads, None, None, None, None, None, None, None)


torch.library.register_autograd("gnop::window_attention", _backward, setup_context=_setup_context, lib=_op_lib)


def _no_second(ctx, *grads):
    raise RuntimeError("window_attention can be differentiated once only")


torch.library.register_autograd("gnop::window_attention_bwd", _no_second, lib=_op_lib)


def _padded(t, D):
    return t if t.shape[-1] == D else F.pad(t, (0, D - t.shape[-1]))


def _attend(q, k, v, lengths, window, sinks, causal, at_end, scale):
    if window is not None and window < 0:
        raise RuntimeError("window must be None or not negative")
    needs = torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v))
    if at_end and needs:
        raise RuntimeError("window_attention_cached has no derivative: call it under torch.no_grad()")
    D = q.shape[-1] if q.dim() else 0
    scale = 1.0 / math.sqrt(max(1, D)) if scale is None else float(scale)
    args = (lengths, -1 if window is None else int(window), int(sinks), bool(causal), at_end, scale, needs)
    if D % 8 == 0 or not q.is_cuda:
        return torch.ops.gnop.window_attention(q, k, v, *args)[0]
    wide = -(-D // 8) * 8  # channels of zeros behind the head add nothing
    return torch.ops.gnop.window_attention(*(_padded(t, wide) for t in (q, k, v)), *args)[0][..., :D]


def window_attention(q, k, v, window=None, sinks=0, causal=False, lengths=None, scale=None):
    """softmax(scale q k^T) v over the tokens that each token sees: those within `window` to either side (None: all), and the
    first `sinks` of its sample, such as registers or a prompt's beginning; none behind it if `causal`.

    q: (B, L, heads, D), k, v: (B, S, kv_heads, D) in float32, float16 or bfloat16, D up to 256 (float32: 128), heads a multiple of kv_heads
    (heads / kv_heads neighbouring heads of q share one of k).  The queries are the last L of the S tokens: L = S is a whole
    sequence, L < S its end.  lengths: (B,) int32 or int64, tokens that a sample has (clamped to 0 .. S): the others are padding,
    which nobody sees, whose rows of the result are zeros, and whose gradients are zeros.  A token that sees nothing gets zeros.
    scale: positive, 1 / sqrt(D) unless given.

    Scores, softmax and sums are in float32, weights are rounded to q's type for the product with v; float32 stays float32
    throughout.  An infinity or a NaN in a token reaches only those that see it.  Slices of one packed projection are read where
    they are; rows that are not whole 16 bytes apart are copied first.  Differentiable once in q, k and v; results and gradients
    are the same bit for bit on every run."""
    if not torch.compiler.is_compiling():
        out = _native.window_attention(q, k, v, lengths, window, sinks, causal, False, scale)
        if out is not NotImplemented:
            return out
    return _attend(q, k, v, lengths, window, sinks, causal, False, scale)


def window_attention_cached(q, k_cache, v_cache, lengths, window=None, sinks=0, scale=None):
    """window_attention of the newest tokens of each request, causal, against caches: for serving.

    q: (B, T, heads, D), k_cache, v_cache: (B, S, kv_heads, D) with room for S tokens, lengths: (B,) int32 or int64, tokens of each
    request that its cache holds (clamped to 0 .. S), the T of q, which are the last of them, included.  What a cache holds behind
    its length has no effect.  A request shorter than T has zeros in front.  It has no derivative."""
    if not torch.compiler.is_compiling():
        out = _native.window_attention(q, k_cache, v_cache, lengths, window, sinks, True, True, scale)
        if out is not NotImplemented:
            return out
    return _attend(q, k_cache, v_cache, lengths, window, sinks, True, True, scale)
