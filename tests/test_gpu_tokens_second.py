"""GPU tests of second derivatives of rms_norm and rotary: through the native calls, through the general form, and of the backward
operators by themselves."""
import pytest
import torch

from gnnhwc import rms_norm, rotary, rotary_frequencies, tokens
from tests import token_refs as ref
from tests.test_gpu_tokens_native import Declining

pytestmark = pytest.mark.gpu
F32, F64, F16, BF16 = torch.float32, torch.float64, torch.float16, torch.bfloat16


@pytest.fixture(params=["native", "general"])
def way(request, monkeypatch):
    if request.param == "general":
        monkeypatch.setattr(tokens, "_native", Declining())


def _normal(shape, dtype, device, seed, mean=0.0):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return (mean + torch.randn(shape, generator=g, dtype=F64)).to(dtype).to(device)


def _leaves(*ts):
    return [t.requires_grad_(True) for t in ts]


# Central differences in float64 of a first derivative: h^2 f'''' / 6 + u f' / h, about 1e-9 at h = 1e-5.
DIFFERENCES = dict(eps=1e-5, atol=1e-7, rtol=1e-6)


def test_norm_against_differences(way, device):
    x, r, w = _leaves(_normal((3, 17), F64, device, 1), _normal((3, 17), F64, device, 2), _normal((17,), F64, device, 3, 1.0))
    check = torch.autograd.gradgradcheck
    assert check(lambda x, r, w: rms_norm(x, w, 1e-3, residual=r, return_sum=True), (x, r, w), **DIFFERENCES)
    assert check(lambda x, r, w: rms_norm(x, w, 1e-3, residual=r), (x, r, w), **DIFFERENCES)  # (its gradients keep the sum)
    assert check(lambda x, w: rms_norm(x, w, 1e-3), (x, w), **DIFFERENCES)
    assert check(lambda x: rms_norm(x, None, 1e-3), (x,), **DIFFERENCES)
    assert check(lambda x: rms_norm(x, w.detach(), 1e-3), (x,), **DIFFERENCES)


@pytest.mark.parametrize("near", [False, True])
def test_rotary_against_differences(way, near, device):
    q, k = _leaves(_normal((2, 3, 2, 12), F64, device, 1), _normal((2, 3, 1, 12), F64, device, 2))
    a, b = _leaves(_normal((12,), F64, device, 3, 1.0), _normal((12,), F64, device, 4, 1.0))
    p, f = torch.tensor([[0, 3], [1, 7], [5, 2]], device=device), rotary_frequencies((2, 3), device=device)
    check = torch.autograd.gradgradcheck
    assert check(lambda q, k, a, b: rotary(q, k, p, f, (2, 3), near, a, b, 1e-3), (q, k, a, b), **DIFFERENCES)
    assert check(lambda q, a: rotary(q, None, p, f, (2, 3), near, a, None, 1e-3), (q, a), **DIFFERENCES)
    assert check(lambda q, k: rotary(q, k, p, f, (2, 3), near), (q, k), **DIFFERENCES)
    assert check(lambda q: rotary(q, None, p, f, (2, 3), near), (q,), **DIFFERENCES)


def _close(got, want, what):
    """The distance of all of a tensor, relative to its size: one rounding, and K float32 ones (tests/token_refs.py) of terms that
    are no more than ten times as large as what they leave."""
    assert got.shape == want.shape, what
    off, size = float((got.double() - want).norm()), float(want.norm())
    assert off <= (ref.U[got.dtype] + 10 * ref.K * ref.U[ref.computing(got.dtype)]) * size, (what, off, size)


def _norm(s, w, eps):
    return s * (s.square().mean(-1, keepdim=True) + eps).rsqrt() * w


@pytest.mark.parametrize("dtype,params", [(F32, F32), (F16, F32), (BF16, BF16)])
def test_backward_of_the_norm_is_differentiable(dtype, params, device):
    s, dy, ds = _leaves(*(_normal((6, 96), dtype, device, i) for i in range(3)))
    w, = _leaves(_normal((96,), params, device, 4, 1.0))
    a, b = _normal((6, 96), dtype, device, 5), _normal((96,), params, device, 6)
    got = torch.autograd.grad(torch.ops.gnop.rms_norm_bwd(dy, ds, s, w, 1e-6), [dy, ds, s, w], [a, b])
    exact = [t.detach().double().requires_grad_(True) for t in (dy, ds, s, w)]
    dx, dw = torch.autograd.grad(_norm(exact[2], exact[3], 1e-6), [exact[2], exact[3]], exact[0], create_graph=True)
    want = torch.autograd.grad([dx + exact[1], dw], exact, [a.double(), b.double()])
    for g, e, name in zip(got, want, ("dy", "ds", "s", "weight")):
        _close(g, e, name)


@pytest.mark.parametrize("near", [False, True])
@pytest.mark.parametrize("dtype,params", [(F32, F32), (F16, F32), (BF16, BF16)])
def test_backward_of_rotary_is_differentiable(dtype, params, near, device):
    sections = (5, 8)
    p, f = torch.randint(0, 50, (7, 2), generator=torch.Generator().manual_seed(1)).to(device), rotary_frequencies((5, 8), device=device)
    d, t = _leaves(_normal((2, 7, 3, 32), dtype, device, 2), _normal((2, 7, 3, 32), dtype, device, 3))
    w, = _leaves(_normal((32,), params, device, 4, 1.0))
    a, b = _normal(d.shape, dtype, device, 5), _normal((32,), params, device, 6)
    out = torch.ops.gnop.rotary_bwd(d, None, t, None, p, f, sections, near, w, None, 1e-6)
    got = torch.autograd.grad([out[0], out[2]], [d, t, w], [a, b])
    exact = [v.detach().double().requires_grad_(True) for v in (d, t, w)]
    angle = ref.angles(p, f, sections)
    first = torch.autograd.grad(ref.turn(_norm(exact[1], exact[2], 1e-6), angle, near), exact[1:], exact[0], create_graph=True)
    want = torch.autograd.grad(first, exact, [a.double(), b.double()])
    for g, e, name in zip(got, want, ("d", "t", "weight")):
        _close(g, e, name)
    # without a norm the gradient is linear in the incoming one
    out = torch.ops.gnop.rotary_bwd(d, None, None, None, p, f, sections, near, None, None, 1e-6)[0]
    assert torch.equal(torch.autograd.grad(out, d, a)[0], torch.ops.gnop.rotary(a, None, p, f, sections, near, None, None, 1e-6)[0])


def test_penalty(way, device):
    """A penalty on the gradient's size, in float32, against the same in elementary operations in float64."""
    x, w = _leaves(_normal((5, 64), F32, device, 1), _normal((64,), F32, device, 2, 1.0))
    p, f = torch.arange(5, device=device), rotary_frequencies((8,), device=device)

    def penalty(x, w, first):
        g, = torch.autograd.grad(first(x, w).pow(3).sum(), x, create_graph=True)
        return torch.autograd.grad((g * g).sum() + (x * x).sum(), [x, w])

    def heads(t):
        return t.view(1, 5, 4, 16)

    got = penalty(x, w, lambda x, w: rotary(heads(rms_norm(x, w)), None, p, f))
    angle = ref.angles(p.view(5, 1), f, (8,))
    want = penalty(x.detach().double().requires_grad_(True), w.detach().double().requires_grad_(True),
                   lambda x, w: ref.turn(heads(_norm(x, w, 1e-6)), angle, False))
    for g, e, name in zip(got, want, ("x", "weight")):
        _close(g, e, name)
