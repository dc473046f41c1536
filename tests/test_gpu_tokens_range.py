"""GPU tests of the backwards of rms_norm and rotary at rows far from one: the root mean square r^-1 of a row may be anything whose
square a float holds, while r^3 leaves a float's range beyond 1e13 and, with eps = 0, below 1e-13.  Bounds: tests/token_refs.py."""
import pytest
import torch

from gnnhwc import rms_norm, rotary, rotary_frequencies
from tests import token_refs as ref

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def _normal(shape, dtype, device, seed, scale=1.0):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return (scale * torch.randn(shape, generator=g, dtype=torch.float64)).to(dtype).to(device)


SIZES = [(1e14, 1e-6), (1e17, 1e-6), (1e-14, 0.0), (1e-17, 0.0)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size,eps", SIZES)
@pytest.mark.parametrize("C", [7, 65, 1024])
def test_norm(C, size, eps, dtype, device):
    x, w = _normal((5, C), dtype, device, 1, size).requires_grad_(True), (1 + 0.2 * _normal((C,), F32, device, 2)).requires_grad_(True)
    if dtype == F32:
        x.data[3] *= 1e-3 if size > 1 else 1e3  # rows of several sizes
    dy = _normal((5, C), dtype, device, 3)
    y = rms_norm(x, w, eps)
    want, _s, scale = ref.rms(x.detach(), w.detach(), eps)
    ref.check(y.detach(), want, scale, "y")
    got = torch.autograd.grad(y, [x, w], dy)
    dx, dx_scale, dw, dw_scale = ref.rms_bwd(dy, None, x.detach(), w.detach(), eps)
    ref.check(got[0], dx, dx_scale, "dx")
    ref.check(got[1], dw, dw_scale, "dw", roundings=ref.K + 32)


@pytest.mark.parametrize("near", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size,eps", SIZES)
def test_heads(size, eps, dtype, near, device):
    B, L, H, D, sections = 2, 9, 3, 64, (12, 16)
    q, w = _normal((B, L, H, D), dtype, device, 1, size).requires_grad_(True), (1 + 0.2 * _normal((D,), F32, device, 2)).requires_grad_(True)
    if dtype == BF16:
        w = w.detach().to(BF16).requires_grad_(True)
    p = torch.randint(0, 500, (L, 2), generator=torch.Generator().manual_seed(3)).to(device)
    f, d = rotary_frequencies(sections, device=device), _normal((B, L, H, D), dtype, device, 4)
    got = torch.autograd.grad(rotary(q, None, p, f, sections, near, q_weight=w, eps=eps), [q, w], d)
    angle = ref.angles(p, f, sections)
    back, pair = ref.turn(d.double(), -angle, near), ref.pair_size(d.double(), angle.shape[-1], near)
    v, u = q.detach().double(), w.detach().double()
    r = 1 / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)
    h, g = v * r, back * u
    want = r * (g - h * (g * h).mean(-1, keepdim=True))
    scale = r * (pair * u.abs() + h.abs() * (pair * u.abs() * h.abs()).mean(-1, keepdim=True))
    ref.check(got[0], want, scale, "dq", roundings=ref.K + 8)
    ref.check(got[1], (back * h).sum((0, 1, 2)), (pair * h.abs()).sum((0, 1, 2)), "dw", roundings=ref.K + 8 + 64)
