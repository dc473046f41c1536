"""Plain float64 forms of the operators for token streams, and the bounds that float32 kernels are held to.

U[t] is half a unit in the last place of type t, relative to a value's magnitude.  A result that is computed in float32 (float64
for float64 data) and rounded once is off by at most U[t] |value| + K u scale, u = U of the computing type, where `scale` is the
magnitude of the terms that were added up and K counts roundings on the way: a row's sum of squares takes at most 8 lane vectors
of 8 values in a lane and 10 steps across lanes, of which the root halves the error, and a result some ten more: K = 64 covers
all of them."""
import torch

U = {torch.float64: 2.0 ** -53, torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
# half the spacing of subnormals (float64's is below every number that is compared here)
LEAST = {torch.float64: 0.0, torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
K = 64


def computing(dtype):
    return torch.float64 if dtype == torch.float64 else torch.float32


def check(got, want, scale, what, roundings=K, dtype=None):
    """|got - want| within the bound above, element by element, both finite; want and scale in float64."""
    dtype = dtype or got.dtype
    got = got.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bound = U[dtype] * want.abs() + LEAST[dtype] + roundings * U[computing(dtype)] * scale
    off = (got - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), "%s: %d of %d off, worst %.3g of its bound, first at %s: %r instead of %r" % (
        what, int(bad.sum()), bad.numel(), float((off / bound)[bad].nan_to_num(float("inf")).max()),
        tuple(int(i) for i in bad.nonzero()[0]), float(got[bad][0]), float(want[bad][0]))


def rms(x, weight, eps, residual=None):
    """(y, s, y's scale) in float64; s is rounded to x's type, as an addition in front of the norm would leave it."""
    s = x if residual is None else (x.double() + residual.double()).to(x.dtype)
    v = s.double()
    h = v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)
    y = h if weight is None else h * weight.double()
    return y, s, y.abs()


def rms_bwd(dy, ds, s, weight, eps):
    """dx, its scale, dw, its scale."""
    v, g = s.double(), dy.double() if weight is None else dy.double() * weight.double()
    r = 1 / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)
    h = v * r
    # (a row's gradient is off by as much as the terms of its mean allow)
    m, m_scale = (g * h).mean(-1, keepdim=True), (g * h).abs().mean(-1, keepdim=True)
    dx, scale = r * (g - h * m), r * (g.abs() + h.abs() * m_scale)
    if ds is not None:
        dx, scale = dx + ds.double(), scale + ds.double().abs()
    t = (dy.double() * h).flatten(0, -2)
    return dx, scale, t.sum(0), t.abs().sum(0)


def angles(positions, frequencies, sections):
    """(B or 1, L, 1, P) in float64."""
    p = positions.double()
    p = p.unsqueeze(0) if p.dim() == 2 else p
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections)).to(p.device)
    return (p[..., axis] * frequencies.double()).unsqueeze(2)


def turn(t, angle, near):
    """t's pairs turned by the angles."""
    P = angle.shape[-1]
    a, b = (t[..., 0:2 * P:2], t[..., 1:2 * P:2]) if near else (t[..., :P], t[..., P:2 * P])
    u, v = a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()
    out = t.clone()
    if near:
        out[..., 0:2 * P:2], out[..., 1:2 * P:2] = u, v
    else:
        out[..., :P], out[..., P:2 * P] = u, v
    return out


def pair_size(t, P, near):
    """Magnitude of the pair that each channel belongs to: what a turned value's error is relative to."""
    a, b = (t[..., 0:2 * P:2], t[..., 1:2 * P:2]) if near else (t[..., :P], t[..., P:2 * P])
    m = a.abs() + b.abs()
    out = t.abs().clone()
    if near:
        out[..., 0:2 * P:2], out[..., 1:2 * P:2] = m, m
    else:
        out[..., :P], out[..., P:2 * P] = m, m
    return out
