"""Dropout of token streams and channels-last features from a counter-based generator: ``dropout``, whose mask is a function of a seed and
an element's place and is never stored, and the module ``Dropout``.  The reference has no counterpart.

The kernel is gnnhwc_dropout of include/gnnhwc_tokens.h.  Ordinary eager calls run in native code (csrc/gn_tokens_torch.cpp); what
that declines comes here, through ``gnop::dropout``, which carries a meta kernel and the autograd formula.
"""
import torch
import torch.nn as nn

from . import _cabi, _native
from .custom_gn import _check_device, _current_stream_ptr, _dtype_code, _on_device, _op_lib


def _signed(n):
    """The 64 bits of an integer, as a signed one."""
    n = int(n) & (2 ** 64 - 1)
    return n - 2 ** 64 if n >= 2 ** 63 else n


def _dropout(x, residual, p, seed, seed_at, offset):
    """gnop::dropout.  Returns y, contiguous.  seed_at: a tensor that holds the seed, or None."""
    _check_device(x, "x")
    dt = _dtype_code(x, "x")
    if residual is not None:
        _check_device(residual, "residual")
        if residual.device != x.device or residual.dtype != x.dtype or residual.shape != x.shape:
            raise RuntimeError("residual must be like x, %s of shape %s on %s" % (x.dtype, tuple(x.shape), x.device))
    if seed_at is not None:
        _check_device(seed_at, "seed")
        if seed_at.device != x.device or seed_at.dtype != torch.int64 or seed_at.numel() != 1:
            raise RuntimeError("a seed tensor must hold one int64 on %s" % x.device)
    if not 0.0 <= p <= 1.0:
        raise RuntimeError("p must be 0 to 1, got %s" % p)
    xc, rc = x.contiguous(), None if residual is None else residual.contiguous()
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    with _on_device(x.device):
        code = _cabi.lib.gnnhwc_dropout(xc.data_ptr(), None if rc is None else rc.data_ptr(), y.data_ptr(), x.numel(), p, seed & (2 ** 64 - 1),
                                        None if seed_at is None else seed_at.data_ptr(), offset & (2 ** 64 - 1), dt, _current_stream_ptr(x.device))
    _cabi.check(code, "gnop::dropout")
    return y


_op_lib.define("dropout(Tensor x, Tensor? residual, float p, int seed, Tensor? seed_at, int offset) -> Tensor")
_op_lib.impl("dropout", _dropout, "CompositeExplicitAutograd")


def _dropout_meta(x, residual, p, seed, seed_at, offset):
    return torch.empty(x.shape, dtype=x.dtype, device=x.device)


_op_lib.impl("dropout", _dropout_meta, "Meta")


def _setup_context(ctx, inputs, output):
    _x, residual, ctx.p, ctx.seed, seed_at, ctx.offset = inputs
    ctx.has_residual = residual is not None
    ctx.save_for_backward(seed_at)


def _backward(ctx, dy):
    seed_at, = ctx.saved_tensors
    dx = torch.ops.gnop.dropout(dy, None, ctx.p, ctx.seed, seed_at, ctx.offset) if ctx.needs_input_grad[0] else None
    return dx, dy if ctx.has_residual else None, None, None, None, None


torch.library.register_autograd("gnop::dropout", _backward, setup_context=_setup_context, lib=_op_lib)


def dropout(x, p, seed, offset=0, residual=None, channel_dim=-1):
    """Each element of x dropped with probability p and otherwise times 1 / (1 - p), plus the residual, in float32 (float64 for float64)
    and rounded to x's type once.

    x: any shape, float32, float64, float16 or bfloat16; residual: a tensor like x, or None.  p is taken in whole multiples of
    2^-16.  The mask is a function of the seed, the offset and an element's place among x's, counted in x's order of dimensions with the one at
    `channel_dim` last (1 for (N, C, H, W), whose channels-last memory is then taken as it is): the same seed and offset give the
    same mask, which is nowhere stored, whatever the layout.  Calls of one seed need an offset each.  seed, offset: integers, of which 64 bits
    count.  seed may also be an int64 tensor with one element on x's device, which is read when the kernel runs: in a captured
    graph, a new seed written there before a replay gives a new mask (forward and backward have to see the same one).

    What is dropped has no effect, an infinity or a NaN neither.  Differentiable in x and residual, as often as need be."""
    if channel_dim != -1 and channel_dim != x.dim() - 1:
        last = [None if t is None else t.movedim(channel_dim, -1) for t in (x, residual)]
        return dropout(last[0], p, seed, offset, last[1]).movedim(-1, channel_dim)
    if not torch.compiler.is_compiling():
        out = _native.dropout(x, residual, p, seed, offset)
        if out is not NotImplemented:
            return out
    at = seed if isinstance(seed, torch.Tensor) else None
    return torch.ops.gnop.dropout(x, residual, float(p), 0 if at is not None else _signed(seed), at, _signed(offset))


class Dropout(nn.Dropout):
    """Module of `dropout`: forward(x) or forward(x, residual), which is residual + dropout(x).  While training, every call draws
    a seed from torch's CPU generator (torch.manual_seed makes it repeatable, and a recomputed forward whose generator state is
    restored draws the same); otherwise x passes, plus the residual.  Where a graph is captured or traced, the seed is a tensor that
    torch's generator of the device fills, with another number at each replay."""

    def __init__(self, p=0.5, channel_dim=-1):
        super().__init__(p)
        self.channel_dim = channel_dim

    def forward(self, x, residual=None):
        if not self.training or self.p == 0.0:
            return x if residual is None else x + residual
        if torch.compiler.is_compiling() or (x.is_cuda and torch.cuda.is_current_stream_capturing()):
            seed = torch.randint(2 ** 63 - 1, (), dtype=torch.int64, device=x.device)
        else:
            seed = int(torch.empty((), dtype=torch.int64, device="cpu").random_())  # (whatever torch's default device is)
        return dropout(x, float(self.p), seed, 0, residual, self.channel_dim)

    def extra_repr(self):
        return "p=%s" % self.p + (", channel_dim=%d" % self.channel_dim if self.channel_dim != -1 else "")
