"""GPU tests of rms_norm and rms_norm_quant against their formulas in float64 (tests/token_refs.py has the bounds and where
they come from)."""
import itertools
import math

import pytest
import torch

from gnnhwc import RMSNorm, rms_norm, rms_norm_quant
from tests import token_refs as ref

pytestmark = pytest.mark.gpu
F32, F64, F16, BF16 = torch.float32, torch.float64, torch.float16, torch.bfloat16
EPS = 1e-6


def _normal(shape, dtype, device, seed, scale=1.0):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return (scale * torch.randn(shape, generator=g, dtype=F64)).to(dtype).to(device)


def _weight(C, dtype, device, seed):
    return (1 + 0.2 * _normal((C,), F64, "cpu", seed)).to(dtype).to(device)


# rows and channels where the cut changes: below a lane vector, odd, one past and one short of full lanes, several wavefronts
SIZES = [(1, 1), (3, 2), (2, 7), (5, 8), (1, 9), (33, 63), (7, 64), (2, 65), (129, 100), (4, 320), (257, 640), (3, 1001), (2, 1280), (5, 2049),
         (2, 2560), (1, 4097), (3, 5120), (2, 8191), (1, 8192)]


@pytest.mark.parametrize("dtype,params", [(F32, F32), (F64, F64), (F16, F16), (F16, F32), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("rows,C", SIZES)
def test_forward_and_backward(rows, C, dtype, params, device):
    for seed, (residual, with_weight) in enumerate(itertools.product((False, True), (False, True))):
        print("rms_norm", rows, C, dtype, params, residual, with_weight, flush=True)
        x = _normal((rows, C), dtype, device, 4 * seed, 2.0).requires_grad_(True)
        r = _normal((rows, C), dtype, device, 4 * seed + 1, 3.0).requires_grad_(True) if residual else None
        w = _weight(C, params, device, 4 * seed + 2).requires_grad_(True) if with_weight else None
        y, s = rms_norm(x, w, EPS, residual=r, return_sum=True)
        want, sum_, scale = ref.rms(x.detach(), None if w is None else w.detach(), EPS, None if r is None else r.detach())
        assert torch.equal(s, sum_)
        ref.check(y.detach(), want, scale, "y")
        with torch.no_grad():
            assert torch.equal(rms_norm(x, w, EPS, residual=r), y)  # the call that keeps no sum
        dy, ds = _normal((rows, C), dtype, device, 50 + seed), _normal((rows, C), dtype, device, 60 + seed)
        inputs = [t for t in (x, r, w) if t is not None]
        got = torch.autograd.grad([y, s] if residual else [y], inputs, [dy, ds] if residual else [dy])
        dx, dx_scale, dw, dw_scale = ref.rms_bwd(dy, ds if residual else None, sum_, None if w is None else w.detach(), EPS)
        ref.check(got[0], dx, dx_scale, "dx")
        if residual:
            assert torch.equal(got[0], got[1])
        if w is not None:
            # terms are off like a forward result; they are added in chains of at most rows / 512 + 32
            ref.check(got[-1], dw, dw_scale, "dw", roundings=ref.K + rows // 512 + 32)


@pytest.mark.parametrize("dtype,C", [(F16, 16384), (BF16, 12289), (F32, 16384), (F32, 10000), (F64, 8192)])
def test_longest_rows(dtype, C, device):
    x, w = _normal((3, C), dtype, device, 1).requires_grad_(True), _weight(C, dtype, device, 2).requires_grad_(True)
    r = _normal((3, C), dtype, device, 3).requires_grad_(True)
    y, s = rms_norm(x, w, EPS, residual=r, return_sum=True)
    want, sum_, scale = ref.rms(x.detach(), w.detach(), EPS, r.detach())
    ref.check(y.detach(), want, scale, "y")
    dy, ds = _normal((3, C), dtype, device, 4), _normal((3, C), dtype, device, 5)
    gx, gw = torch.autograd.grad([y, s], [x, w], [dy, ds])
    dx, dx_scale, dw, dw_scale = ref.rms_bwd(dy, ds, sum_, w.detach(), EPS)
    ref.check(gx, dx, dx_scale, "dx")
    ref.check(gw, dw, dw_scale, "dw", roundings=ref.K + 32)


@pytest.mark.parametrize("rows,C", [(5000, 96), (20011, 40), (2048, 1280)])
def test_many_rows(rows, C, device):
    x, w = _normal((rows, C), BF16, device, 1).requires_grad_(True), _weight(C, F32, device, 2).requires_grad_(True)
    dy = _normal((rows, C), BF16, device, 3)
    y = rms_norm(x, w, EPS)
    first = torch.autograd.grad(y, [x, w], dy, retain_graph=True)
    second = torch.autograd.grad(y, [x, w], dy)
    assert all(torch.equal(a, b) for a, b in zip(first, second))  # the order of sums is fixed
    dx, dx_scale, dw, dw_scale = ref.rms_bwd(dy, None, x.detach(), w.detach(), EPS)
    ref.check(first[0], dx, dx_scale, "dx")
    ref.check(first[1], dw, dw_scale, "dw", roundings=ref.K + rows // 512 + 32)


def test_gradients_against_differences(device):
    """Central differences in float64: error of the difference h^2 f'''/6 + u f / h, at h = 1e-5 about 1e-9 here."""
    x, r, w = _normal((4, 37), F64, device, 1), _normal((4, 37), F64, device, 2), _weight(37, F64, device, 3)
    for t in (x, r, w):
        t.requires_grad_(True)
    assert torch.autograd.gradcheck(lambda *a: rms_norm(a[0], a[2], 1e-3, residual=a[1], return_sum=True), (x, r, w), eps=1e-5, atol=1e-7, rtol=1e-6)
    assert torch.autograd.gradcheck(lambda a: rms_norm(a, None, 1e-3), (x,), eps=1e-5, atol=1e-7, rtol=1e-6)


def test_one_output_of_two(device):
    """Only y, or only the sum, reaches the loss."""
    x, r = _normal((6, 48), F32, device, 1).requires_grad_(True), _normal((6, 48), F32, device, 2).requires_grad_(True)
    w = _weight(48, F32, device, 3).requires_grad_(True)
    y, s = rms_norm(x, w, EPS, residual=r, return_sum=True)
    g = _normal((6, 48), F32, device, 4)
    only_y = torch.autograd.grad(y, [x, r], g, retain_graph=True)
    dx, scale, _dw, _ = ref.rms_bwd(g, None, s.detach(), w.detach(), EPS)
    ref.check(only_y[0], dx, scale, "dx")
    only_s = torch.autograd.grad(s, [x, r], g)
    assert torch.equal(only_s[0], g) and torch.equal(only_s[1], g)
    # the sum is not asked for, and gradients are: it is kept for the backward all the same
    y = rms_norm(x, w, EPS, residual=r)
    assert torch.equal(torch.autograd.grad(y, x, g)[0], only_y[0])


def test_layouts(device):
    """Slices, transposed and channels-last tensors give what their contiguous copies give."""
    C = 72
    wide = _normal((6, 5, 3 * C), BF16, device, 1)
    w = _weight(C, BF16, device, 2)
    for name, t in (("slice", wide[..., C:2 * C]), ("odd offset", wide[..., 1:1 + C]), ("every other row", wide[::2, :, :C]),
                    ("transposed rows", wide[..., :C].transpose(0, 1)), ("expanded", wide[:1, :1, :C].expand(6, 5, C)),
                    ("channels apart", wide[..., ::3])):
        assert torch.equal(rms_norm(t, w, EPS), rms_norm(t.contiguous(), w, EPS)), name
    image = _normal((2, C, 7, 5), BF16, device, 3).to(memory_format=torch.channels_last)
    rows = image.permute(0, 2, 3, 1).contiguous()
    y = rms_norm(image, w, EPS, channel_dim=1)
    assert y.shape == image.shape and y.stride(1) == 1
    assert torch.equal(y.permute(0, 2, 3, 1), rms_norm(rows, w, EPS))
    y, s = RMSNorm(C, channel_dim=1).to(device).bfloat16()(image, image)
    assert y.shape == s.shape == image.shape and torch.equal(s, image + image)
    # a residual that is one row for all: its gradient is the sum over them (autograd's own)
    x, r = _normal((9, C), F32, device, 4).requires_grad_(True), _normal((1, C), F32, device, 5).requires_grad_(True)
    y = rms_norm(x, None, EPS, residual=r.expand(9, C))
    gx, gr = torch.autograd.grad(y, [x, r], torch.ones_like(y))
    assert gr.shape == (1, C) and torch.allclose(gr, gx.sum(0, keepdim=True), rtol=1e-5, atol=1e-5)


def test_values_at_the_edges(device):
    """Rows of zeros, of the largest and the smallest values, with infinities and NaN: what the formula gives, and only in their row."""
    C = 130
    for dtype in (F32, F16, BF16):
        x = _normal((7, C), dtype, device, 1)
        x[1] = 0
        x[2] = torch.finfo(dtype).smallest_normal
        x[3] = 1e4
        x[4, 5] = math.inf
        x[5, 129] = math.nan
        y = rms_norm(x, None, EPS)
        want, _s, scale = ref.rms(x, None, EPS)
        fine = [0, 1, 2, 3, 6]
        ref.check(y[fine], want[fine], scale[fine], "y")
        assert torch.equal(y[4].isnan(), torch.arange(C, device=device) == 5) and (y[4].nan_to_num(0) == 0).all()
        assert y[5].isnan().all()
        g = torch.ones_like(x)
        x.requires_grad_(True)
        dx, = torch.autograd.grad(rms_norm(x, None, EPS), x, g)
        want, scale, _dw, _ = ref.rms_bwd(g, None, x.detach(), None, EPS)
        ref.check(dx[fine], want[fine], scale[fine], "dx")
        assert dx[5].isnan().all()


def test_empty_rows(device):
    w = torch.ones(16, device=device, requires_grad=True)
    x = torch.zeros((0, 3, 16), device=device, requires_grad=True)
    y, s = rms_norm(x, w, EPS, residual=torch.zeros_like(x), return_sum=True)
    assert y.shape == s.shape == x.shape
    dx, dw = torch.autograd.grad(y, [x, w], torch.zeros_like(y))
    assert dx.shape == x.shape and torch.equal(dw, torch.zeros_like(w))


def test_other_stream_and_graph(device):
    x, w, r = _normal((64, 640), BF16, device, 1), _weight(640, BF16, device, 2), _normal((64, 640), BF16, device, 3)
    want = rms_norm(x, w, EPS, residual=r, return_sum=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = rms_norm(x, w, EPS, residual=r, return_sum=True)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    xs, ws = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    dy = _normal((64, 640), BF16, device, 4)

    def step():
        y = rms_norm(xs, ws, EPS, residual=r)
        grads = torch.autograd.grad(y, [xs, ws], dy)
        return (y.detach(), *grads, *rms_norm_quant(xs.detach(), ws.detach(), EPS))

    with torch.cuda.stream(side):
        for _ in range(3):
            step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in range(3):
        xs.data.copy_(_normal((64, 640), BF16, device, 10 + seed))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, step()):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_compiled_whole(device):
    x, r = _normal((8, 96), F32, device, 1).requires_grad_(True), _normal((8, 96), F32, device, 2)
    w = _weight(96, F32, device, 3).requires_grad_(True)

    def f(x, w, r):
        y, s = rms_norm(x, w, EPS, residual=r, return_sum=True)
        return (y * y).sum() + s.sum()

    want = torch.autograd.grad(f(x, w, r), [x, w])
    got = torch.autograd.grad(torch.compile(f, backend="aot_eager", fullgraph=True)(x, w, r), [x, w])
    for a, b in zip(got, want):
        assert torch.equal(a, b)


# ---- 8 bits ----------------------------------------------------------------------------------------------------------
QMOST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def _quantised(y, block, out):
    """(values in units of the scale, scales) in float64."""
    C = y.shape[-1]
    block = block or C
    parts = y.split(block, dim=-1)
    scales = torch.stack([(p.abs().amax(-1) / QMOST[out]).clamp(min=2.0 ** -126) for p in parts], -1)
    return torch.cat([p / s.unsqueeze(-1) for p, s in zip(parts, scales.unbind(-1))], -1), scales


def _check_quantised(q, scales, y, block, out):
    units, want = _quantised(y, block, out)
    ref.check(scales, want, want.abs(), "scales")
    # a value is off by half a step (e4m3: 2^-4 of its magnitude, at least 2^-10; integers: 1/2) and by the float32 error
    off = (q.double() - units).abs()
    step = (units.abs() * 2.0 ** -4).clamp(min=2.0 ** -10) if out == torch.float8_e4m3fn else torch.full_like(units, 0.5)
    assert (off <= step + 2 * ref.K * 2.0 ** -24 * units.abs()).all(), float((off - step).max())
    assert float(q.double().abs().max()) <= QMOST[out]


@pytest.mark.parametrize("out", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("dtype,params", [(F32, F32), (F16, F16), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize("rows,C,block", [(1, 1, None), (2, 7, None), (3, 64, 16), (5, 100, 32), (4, 129, 128), (33, 320, 64), (2, 1001, 256),
                                          (7, 1111, None), (3, 1280, 128), (2, 2560, 256), (1, 5120, None), (2, 8192, 128), (1, 16384, 256),
                                          (257, 40, 64), (9, 333, 16)])
def test_quantised(rows, C, block, dtype, params, out, device):
    print("rms_norm_quant", rows, C, block, dtype, params, out, flush=True)
    x, w = _normal((rows, C), dtype, device, 1, 2.0), _weight(C, params, device, 2)
    r = _normal((rows, C), dtype, device, 3)
    x[0, C // 2] *= 30  # an outlier
    for residual in (None, r):
        q, scales, s = rms_norm_quant(x, w, EPS, residual=residual, return_sum=True, out_dtype=out, block=block)
        y, sum_, _ = ref.rms(x, w, EPS, residual)
        assert q.dtype == out and q.shape == x.shape and torch.equal(s, sum_)
        assert scales.shape == (rows, -(-C // block) if block and block < C else 1) and scales.dtype == F32
        _check_quantised(q, scales, y, block if block and block < C else None, out)
        two = rms_norm_quant(x, w, EPS, residual=residual, out_dtype=out, block=block)
        assert len(two) == 2 and torch.equal(two[0].view(torch.uint8), q.view(torch.uint8)) and torch.equal(two[1], scales)


def test_quantised_edges(device):
    x = _normal((6, 256), BF16, device, 1)
    x[1] = 0
    x[2, 3] = math.nan
    x[3, 200] = math.inf
    x[4] = 1e-38  # far below eps: y is denormal in part
    for out in QMOST:
        q, scales = rms_norm_quant(x, None, EPS, out_dtype=out, block=128)
        assert (q[1].float() == 0).all() and (scales[1] == 2.0 ** -126).all()
        assert scales[2].isnan().all() and scales[3, 1].isnan() and scales[3, 0] == 2.0 ** -126
        assert scales[[0, 1, 4, 5]].isfinite().all()
        if out == torch.float8_e4m3fn:
            assert q[2].float().isnan().all() and q[3, 128:].float().isnan().all() and (q[3, :128].float() == 0).all()
        fine = [0, 4, 5]
        _check_quantised(q[fine], scales[fine], ref.rms(x[fine], None, EPS)[0], 128, out)
    q, scales = rms_norm_quant(torch.zeros((0, 64), device=device), None)
    assert q.shape == (0, 64) and scales.shape == (0, 1)


def test_refusals(device):
    x, w = torch.zeros((2, 8), device=device), torch.ones(8, device=device)
    for call, text in ((lambda: rms_norm(x, w[:4]), "8 elements"), (lambda: rms_norm(x, w.half()), "weight must be"),
                       (lambda: rms_norm(x, w.cpu()), "must be a CUDA tensor"), (lambda: rms_norm(x.cpu(), w), "must be a CUDA tensor"),
                       (lambda: rms_norm(x.int(), None), "not implemented"), (lambda: rms_norm(x, w, residual=x[:1]), "residual must be"),
                       (lambda: rms_norm(x, w, residual=x.half()), "residual must be"), (lambda: rms_norm(x, w, -1.0), "eps"),
                       (lambda: rms_norm(torch.zeros((1, 20000), device=device)), "channels"),
                       (lambda: rms_norm(torch.zeros((1, 9000), device=device, dtype=F64)), "channels"),
                       (lambda: rms_norm(torch.zeros((3, 0), device=device)), "shape"),
                       (lambda: rms_norm_quant(x, w, out_dtype=F16), "out_dtype"), (lambda: rms_norm_quant(x.double()), "8-bit"),
                       (lambda: rms_norm_quant(torch.zeros((1, 600), device=device), block=100), "block"),
                       (lambda: rms_norm_quant(torch.zeros((1, 600), device=device), block=512), "block"),
                       (lambda: rms_norm_quant(torch.zeros((1, 600), device=device), block=0), "block"),
                       (lambda: rms_norm_quant(x.clone().requires_grad_(True), w), "no derivative")):
        with pytest.raises(RuntimeError, match=text):
            call()
