"""Plain float64 attention with a window and sinks, and the bounds that the kernels' results are held to, element by element.

u is half a unit of float32, U half a unit of the tensors' type, and a sum of n float32 terms t is off by at most n u sum |t| (the
kernels add them in chains of n / 16 or fewer, so that this is ample).  With e the largest error of a score in powers of two,
  e = (D + 4) u scale log2(e) sum_d |q_d k_d| + 4 u (|score| + |lse|),
a weight w is off by w (ln 2 * 2 e + 8 u): its exponential, and the sum that it is divided by.  As an operand it is rounded once
more: U w, and in float16 at least half the spacing of subnormals, 2^-25 of the largest weight's order (weights are held below
2^8 and the sum of weights is 1 or more; in the backward as 2^12 w).
  out:  sum_j |v_j| (error of w_j)                                                  + U |out|
  dv:   sum_i |do_i| (error of w_ij)                                                + U |dv|
  dS:   the error of w times |dP - delta|, w times those of dP (D + 4) u sum |do v| and of delta (U^2 + 3 (D + 4) u) sum |do o| (which
        comes from the rounded out and from what rounding left of it, itself rounded: off by U^2, in float16 by half a subnormal or more), and U dS for its own rounding; in float16 2^-25 of the unit: |dS| is held as 32 dS /
        (largest |do|), within a factor of two
  dq:   scale sum_j |k_j| (error of dS_ij) + U |dq|,   dk: scale sum_i |q_i| (error of dS_ij) + U |dk|
and the float32 sums of the second products add (n / 16 + 64) u of the magnitudes that they add up."""
import math

import torch

from tests.token_refs import LEAST, U

u = U[torch.float32]


def sees(B, L, S, window, sinks, causal, lengths, at_end, device):
    """(B, L, S) truth values: which tokens each query sees, by the definition."""
    n = torch.full((B,), S, device=device) if lengths is None else lengths.to(device).long().clamp(0, S)
    n = n.view(B, 1, 1)
    p = torch.arange(L, device=device).view(1, L, 1) + (n if at_end else S) - L
    j = torch.arange(S, device=device).view(1, 1, S)
    near = torch.ones((B, L, S), dtype=torch.bool, device=device) if window is None else (j - p).abs() <= window
    seen = (near | (j < sinks)) & (j < n) & (p >= 0) & (p < n)
    return seen & (j <= p) if causal else seen


def _heads(t, K):
    """(B, L, H, D) -> (B, K, G, L, D) in float64."""
    return t.detach().double().unflatten(2, (K, t.shape[2] // K)).permute(0, 2, 3, 1, 4)


def _back(t):
    """(B, K, G, L, D) -> (B, L, K G, D)."""
    return t.permute(0, 3, 1, 2, 4).flatten(2, 3)


def attention(q, k, v, seen, scale, dout=None):
    """{name: (value, bound)} of out and, with dout, of dq, dk and dv, in float64.  Tokens that nobody sees may hold anything."""
    B, L, H, D = q.shape
    S, K = k.shape[1], k.shape[2]
    dtype = q.dtype
    least = LEAST[dtype] if dtype == torch.float16 else 0.0
    m = seen.view(B, 1, 1, L, S)
    row = seen.any(2).view(B, L, 1, 1)
    col = seen.any(1).view(B, S, 1, 1)
    Q, Kd, V = _heads(q.detach().where(row, torch.zeros((), dtype=dtype, device=q.device)), K), \
        _heads(k.detach().where(col, torch.zeros((), dtype=dtype, device=q.device)), K), \
        _heads(v.detach().where(col, torch.zeros((), dtype=dtype, device=q.device)), K)
    s = scale * Q @ Kd.transpose(-1, -2)
    s = s.masked_fill(~m, -math.inf)
    most = s.amax(-1, keepdim=True)
    most = most.masked_fill(most == -math.inf, 0.0)
    w = (s - most).exp()
    total = w.sum(-1, keepdim=True)
    w = w / total.masked_fill(total == 0, 1.0)
    lse = ((total.masked_fill(total == 0, 1.0)).log() + most) / math.log(2)
    out = w @ V
    size = scale * math.log2(math.e) * (Q.abs() @ Kd.abs().transpose(-1, -2))
    e = (D + 4) * u * size + 4 * u * (size + lse.abs())
    e = (e * m).amax(-1, keepdim=True)
    off = w * (2 * math.log(2) * e + 8 * u)
    summed = (S / 16 + 64) * u
    rounded = U[dtype] if dtype != torch.float32 else 0.0
    w_off = (off + rounded * w + least * m)
    result = {"out": (_back(out), _back((w_off + summed * w) @ V.abs() + U[dtype] * out.abs() + LEAST[dtype]))}
    if dout is None:
        return result
    G = _heads(dout.detach().where(row, torch.zeros((), dtype=dtype, device=q.device)), K)

    def shared(t):
        return t.sum(2, keepdim=True)

    dv = shared(w.transpose(-1, -2) @ G)
    dv_off = shared((w_off + (H // K) * summed * w).transpose(-1, -2) @ G.abs())
    dp, delta = G @ V.transpose(-1, -2), (G * out).sum(-1, keepdim=True)
    ds = w * (dp - delta)
    unit = G.abs().amax()
    d_off = off * (dp - delta).abs() + w * ((D + 4) * u * (G.abs() @ V.abs().transpose(-1, -2)) + (rounded ** 2 + 3 * (D + 4) * u) * (G.abs() * out.abs()).sum(-1, keepdim=True)
                                              + least * G.abs().sum(-1, keepdim=True))
    # (out's own error, as far as delta is made of it)
    d_off = d_off + w * (G.abs() * ((w_off + summed * w) @ V.abs())).sum(-1, keepdim=True)
    d_off = (d_off + rounded * (ds.abs() + d_off) + least * unit / 16 * m) * m
    dq, dk = scale * ds @ Kd, shared(scale * ds.transpose(-1, -2) @ Q)
    dq_off = scale * (d_off + summed * ds.abs()) @ Kd.abs()
    dk_off = shared(scale * (d_off + (H // K) * summed * ds.abs()).transpose(-1, -2) @ Q.abs())
    for name, value, bound in (("dq", dq, dq_off), ("dk", dk, dk_off), ("dv", dv, dv_off)):
        result[name] = (_back(value), _back(bound + U[dtype] * (value.abs() + bound) + LEAST[dtype]))
    return result


def check(got, want, what):
    """Every element within its bound."""
    value, bound = want
    got = got.detach().double()
    assert got.shape == value.shape, (what, got.shape, value.shape)
    off = (got - value).abs()
    bad = ~(off <= bound)
    assert not bad.any(), "%s: %d of %d off, worst %.3g of its bound, first at %s: %r instead of %r (bound %.3g)" % (
        what, int(bad.sum()), bad.numel(), float((off / bound)[bad].nan_to_num(float("inf")).max()), tuple(int(i) for i in bad.nonzero()[0]),
        float(got[bad][0]), float(value[bad][0]), float(bound[bad][0]))
