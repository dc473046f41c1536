"""GPU tests of the operators for token streams on tensors that no cache holds (more than 224 MiB of inputs), which kernels of their
own read past the caches: every element against the float64 formulas, a stretch of rows at a time."""
import math

import pytest
import torch

from gnnhwc import clip_gradients, rms_norm, rms_norm_quant, rotary, rotary_frequencies
from tests import token_refs as ref
from tests.test_gpu_rms import _check_quantised

pytestmark = pytest.mark.gpu
F32, F64, F16, BF16 = torch.float32, torch.float64, torch.float16, torch.bfloat16
EPS = 1e-6
CACHED = 224 << 20


@pytest.fixture(autouse=True)
def _free():
    yield
    torch.cuda.empty_cache()


def _normal(shape, dtype, device, seed, scale=1.0):
    g = torch.Generator(device=device).manual_seed(seed)
    return torch.empty(shape, dtype=dtype, device=device).normal_(generator=g).mul_(scale)


def _weight(C, dtype, device, seed):
    return (1 + 0.2 * _normal((C,), F32, device, seed)).to(dtype)


@pytest.mark.parametrize("rows,C,dtype,params", [(50_001, 2560, BF16, F32), (26_003, 2560, F32, F32), (7_500, 16384, F16, F16), (130_003, 1000, BF16, BF16),
                                                 (4_100, 8192, F64, F64)])
@pytest.mark.parametrize("residual", [False, True])
def test_norm(rows, C, dtype, params, residual, device):
    print("rms_norm", rows, C, dtype, params, residual, flush=True)
    x, w = _normal((rows, C), dtype, device, 1, 2.0).requires_grad_(True), _weight(C, params, device, 2).requires_grad_(True)
    r = _normal((rows, C), dtype, device, 3, 3.0).requires_grad_(True) if residual else None
    assert x.numel() * x.element_size() > CACHED
    dy, ds = _normal((rows, C), dtype, device, 4), _normal((rows, C), dtype, device, 5) if residual else None
    y, s = rms_norm(x, w, EPS, residual=r, return_sum=True)
    dx, dw = torch.autograd.grad([y, s] if residual else [y], [x, w], [dy, ds] if residual else [dy])
    x, r, w, y, s = (None if t is None else t.detach() for t in (x, r, w, y, s))
    step, want_dw, dw_scale = max(1, (1 << 24) // C), 0, 0
    for at in range(0, rows, step):
        part = slice(at, min(rows, at + step))
        want, sum_, scale = ref.rms(x[part], w, EPS, r[part] if residual else None)
        assert torch.equal(s[part], sum_), at
        ref.check(y[part], want, scale, "y from row %d" % at)
        want, scale, a, b = ref.rms_bwd(dy[part], ds[part] if residual else None, sum_, w, EPS)
        ref.check(dx[part], want, scale, "dx from row %d" % at)
        want_dw, dw_scale = want_dw + a, dw_scale + b
    ref.check(dw, want_dw, dw_scale, "dw", roundings=ref.K + rows // 512 + 32)


@pytest.mark.parametrize("out", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("rows,C,block,dtype,residual", [(60_001, 2560, 128, BF16, False), (50_003, 2560, None, F16, True), (40_000, 1664, 256, F32, True),
                                                         (9_000, 16384, 64, BF16, False)])
def test_quantised(rows, C, block, dtype, residual, out, device):
    x, w = _normal((rows, C), dtype, device, 1, 2.0), _weight(C, F32, device, 2)
    r = _normal((rows, C), dtype, device, 3) if residual else None
    assert x.numel() * x.element_size() > CACHED
    q, scales, s = rms_norm_quant(x, w, EPS, residual=r, return_sum=True, out_dtype=out, block=block)
    for at in range(0, rows, 5000):
        part = slice(at, min(rows, at + 5000))
        y, sum_, _ = ref.rms(x[part], w, EPS, r[part] if residual else None)
        assert torch.equal(s[part], sum_), at
        _check_quantised(q[part], scales[part], y, block, out)


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("near", [False, True])
@pytest.mark.parametrize("L,H,K,D,dtype", [(40_003, 24, 24, 64, BF16), (30_001, 24, 8, 128, F16), (30_001, 20, 12, 64, F32), (20_003, 6, 4, 160, F64)])
def test_rotary(L, H, K, D, dtype, near, norm, device):
    print("rotary", L, H, K, D, dtype, near, norm, flush=True)
    packed = _normal((1, L, (H + 2 * K) * D), dtype, device, 1)
    q, k = packed[..., :H * D].view(1, L, H, D).detach().requires_grad_(True), packed[..., H * D:(H + K) * D].view(1, L, K, D).detach().requires_grad_(True)
    assert L * (H + K) * D * q.element_size() > CACHED
    sections = (D // 8, D // 2 - D // 8)
    w = [_weight(D, dtype, device, 2 + i).requires_grad_(True) if norm else None for i in range(2)]
    p, f = torch.stack([torch.arange(L, device=device) % 199, torch.arange(L, device=device)], dim=-1), rotary_frequencies(sections, device=device)
    outs = rotary(q, k, p, f, sections, near, *w, EPS)
    given = _normal(q.shape, dtype, device, 4), _normal(k.shape, dtype, device, 5)
    inputs = [q, k] + [t for t in w if t is not None]
    back = torch.autograd.grad(outs, inputs, given)
    roundings = 8 + (ref.K if norm else 0)  # (a turned pair, and the norm in front of it: tests/test_gpu_rotary.py)
    for side in range(2):
        t, out, d, dt, u = inputs[side].detach(), outs[side].detach(), given[side], back[side], w[side]
        u = None if u is None else u.detach().double()
        want_dw, dw_scale = 0, 0
        for at in range(0, L, 4000):
            part = slice(at, min(L, at + 4000))
            angle = ref.angles(p[part], f, sections)
            v, g = t[:, part].double(), ref.turn(d[:, part].double(), -angle, near)
            size = ref.pair_size(d[:, part].double(), angle.shape[-1], near)
            if norm:
                r = 1 / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS)
                h = v * r
                want_dw, dw_scale = want_dw + (g * h).sum((0, 1, 2)), dw_scale + (size * h.abs()).sum((0, 1, 2))
                scale = r * (size * u.abs() + h.abs() * (size * u.abs() * h.abs()).mean(-1, keepdim=True))
                g = r * (g * u - h * (g * u * h).mean(-1, keepdim=True))
                v, size = h * u, scale
            ref.check(out[:, part], ref.turn(v, angle, near), ref.pair_size(v, angle.shape[-1], near), "qk"[side], roundings)
            ref.check(dt[:, part], g, size, "d" + "qk"[side], roundings)
        if norm:
            ref.check(back[2 + side], want_dw, dw_scale, "dw of " + "qk"[side], roundings + L * t.shape[2] // 512 + 96)


@pytest.mark.parametrize("dtype,out", [(BF16, F32), (F16, F16), (F32, BF16), (F64, F32), (BF16, None), (F32, None), (F64, None)])
def test_clipping(dtype, out, device):
    sizes = [60_000_001, 16_384, 333, 70_000_000, 5]
    grads = [_normal((n,), dtype, device, i, 1e-3) for i, n in enumerate(sizes)]
    assert sum(n * g.element_size() for n, g in zip(sizes, grads)) > CACHED
    before = [g.clone() for g in grads]
    to = None if out is None else [torch.full((n,), 7.0, dtype=out, device=device) for n in sizes]
    total = clip_gradients(grads, 2.5, out=to)
    want = math.sqrt(sum(float(p.double().square().sum()) for g in before for p in g.split(1 << 24)))
    u = ref.U[total.dtype]
    assert abs(float(total) - want) <= 4 * u * want + 1e-14 * want
    factor = 2.5 / (want + 1e-6)
    for i, (g, o) in enumerate(zip(before, grads if out is None else to)):
        for a, b in zip(g.split(1 << 24), o.split(1 << 24)):
            ref.check(b, a.double() * factor, (a.double() * factor).abs(), "result %d" % i, roundings=16)
    if out is not None:
        assert all(torch.equal(a, b) for a, b in zip(before, grads))
