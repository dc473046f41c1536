"""GPU tests of clip_gradients and clip_grad_norm_ against their formula in float64.

The norm is a sum of squares in float64, so that it is off by the rounding to float32 alone (2 u with the last steps); a factor
by three more; a result by one product and one rounding."""
import math

import pytest
import torch

from gnnhwc import clip_grad_norm_, clip_gradients
from tests import token_refs as ref

pytestmark = pytest.mark.gpu
F32, F64, F16, BF16 = torch.float32, torch.float64, torch.float16, torch.bfloat16


def _grads(shapes, dtypes, device, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(scale * torch.randn(s, generator=g, dtype=F64)).to(d).to(device) for s, d in zip(shapes, dtypes)]


def _norm(grads):
    return math.sqrt(sum(float(g.double().square().sum()) for g in grads))


def _check_total(total, want):
    u = ref.U[total.dtype]
    assert total.dim() == 0 and abs(float(total) - want) <= 4 * u * want + (1e-14 * want if u < 1e-10 else 0), (float(total), want)


def _check_scaled(got, grads, factor):
    for i, (o, g) in enumerate(zip(got, grads)):
        want = g.double() * factor
        ref.check(o, want, want.abs(), "result %d" % i, roundings=8 if o.dtype != F64 else 16)


SHAPES = [(1,), (7,), (64, 3, 3, 3), (8191,), (8192,), (8193,), (3, 0, 2), (320, 320), (5, 1, 77), (24577,), ()]


@pytest.mark.parametrize("dtypes", [(F32,), (F64,), (F16,), (BF16,), (F32, BF16, F16, F64)])
@pytest.mark.parametrize("max_norm", [0.5, 1e6])
def test_in_place_and_elsewhere(dtypes, max_norm, device):
    types = [dtypes[i % len(dtypes)] for i in range(len(SHAPES))]
    grads = _grads(SHAPES, types, device, 1)
    before, want = [g.clone() for g in grads], _norm(grads)
    for out_types in (types, [F32] * len(SHAPES), [dtypes[(i + 1) % len(dtypes)] for i in range(len(SHAPES))]):
        out = [torch.full(s, 7.0, dtype=d, device=device) for s, d in zip(SHAPES, out_types)]
        total = clip_gradients(grads, max_norm, out=out)
        assert total.dtype == (F64 if set(types) == {F64} else F32)
        _check_total(total, want)
        _check_scaled(out, before, min(1.0, max_norm / (want + 1e-6)))
        assert all(torch.equal(a, b) for a, b in zip(grads, before))
    _check_total(clip_gradients(grads, max_norm), want)
    _check_scaled(grads, before, min(1.0, max_norm / (want + 1e-6)))
    if max_norm > want:
        assert all(torch.equal(a, b) for a, b in zip(grads, before))


@pytest.mark.parametrize("count,size", [(1, 3_000_001), (500, 97), (260, 8200), (113, 1), (112, 5), (1300, 65)])
def test_many_and_large(count, size, device):
    """More tensors than one table holds; gradients far apart in memory and neighbours in a bucket."""
    for packed in (False, True):
        if packed:
            bucket = _grads([(count * size + 3,)], [BF16], device, 2)[0]
            grads = [bucket[1 + i * size:1 + (i + 1) * size] for i in range(count)]
            edges = bucket[[0, -2, -1]].clone()
        else:
            grads = _grads([(size,)] * count, [BF16] * count, device, 2)
        before, want = [g.clone() for g in grads], _norm(grads)
        out = [torch.empty(size, device=device) for _ in range(count)]
        _check_total(clip_gradients(grads, 1.5, out=out), want)
        _check_scaled(out, before, 1.5 / (want + 1e-6))
        first = clip_gradients(grads, 1.5)
        _check_total(first, want)
        _check_scaled(grads, before, 1.5 / (want + 1e-6))
        if packed:
            assert torch.equal(bucket[[0, -2, -1]], edges)


def test_reproducible(device):
    grads = _grads([(100_003,), (4097, 33)], [F32, F32], device, 3)
    totals = {float(clip_gradients(grads, math.inf)) for _ in range(5)}
    assert len(totals) == 1


def test_range(device):
    """Squares beyond the range of a float, at both ends."""
    for scale in (1e25, 1e-30):
        grads = [torch.full((1000,), scale, device=device), torch.full((24,), scale, device=device, dtype=BF16)]
        want = _norm(grads)
        before = [g.clone() for g in grads]
        _check_total(clip_gradients(grads, 0.25 * scale), want)
        _check_scaled(grads, before, 0.25 * scale / (want + 1e-6))


def test_scale(device):
    """Gradients of a scaled loss: the norm and the bound are those of the unscaled ones."""
    grads = _grads([(1000,), (33, 7)], [F16, F16], device, 4, scale=64.0)
    want = _norm(grads) / 1024
    out = [torch.empty_like(g, dtype=F32) for g in grads]
    _check_total(clip_gradients(grads, 0.1, out=out, grad_scale=1 / 1024), want)
    _check_scaled(out, grads, 0.1 / (want + 1e-6) / 1024)
    _check_total(clip_gradients(grads, math.inf, out=out, grad_scale=-1 / 1024), want)
    _check_scaled(out, grads, -1 / 1024)


def test_infinite_and_nan(device):
    grads = _grads([(100,), (50,)], [F32, F32], device, 5)
    grads[0][3] = math.inf
    total = clip_gradients(grads, 1.0)
    assert float(total) == math.inf and grads[0][3].isnan() and (grads[1] == 0).all()
    grads = _grads([(100,), (50,)], [F32, F32], device, 5)
    grads[1][49] = math.nan
    before = grads[0].clone()
    assert math.isnan(float(clip_gradients(grads, math.inf))) and torch.equal(grads[0], before)  # the norm only
    assert math.isnan(float(clip_gradients(grads, 1.0))) and grads[0].isnan().all()
    zeros = [torch.zeros(9, device=device)]
    assert float(clip_gradients(zeros, 1.0)) == 0 and (zeros[0] == 0).all()


def test_layouts(device):
    w = _grads([(8, 4, 3, 3)], [F32], device, 6)[0].to(memory_format=torch.channels_last)
    wide = _grads([(10, 12)], [F32], device, 7)[0]
    slice_, t = wide[:, 2:9], _grads([(5, 6)], [F32], device, 8)[0].t()
    grads = [w, slice_, t]
    before, want = [g.clone() for g in grads], _norm(grads)
    rest = wide[:, [0, 1, 9, 10, 11]].clone()
    out = [torch.empty_like(w), torch.empty(10, 7, device=device), torch.empty(6, 5, device=device)]
    _check_total(clip_gradients(grads, 2.0, out=out), want)
    _check_scaled(out, before, 2.0 / (want + 1e-6))
    strided = [torch.empty(8, 4, 3, 3, device=device), torch.empty(10, 14, device=device)[:, ::2], torch.empty(5, 6, device=device).t()]
    clip_gradients(grads, 2.0, out=strided)
    assert all(torch.equal(a, b) for a, b in zip(strided, out))
    _check_total(clip_gradients(grads, 2.0), want)
    _check_scaled(grads, before, 2.0 / (want + 1e-6))
    assert torch.equal(wide[:, [0, 1, 9, 10, 11]], rest)


def test_negated_views(device):
    """The imaginary part of a conjugate is a view whose memory holds the negated values."""
    z = torch.complex(*_grads([(50,), (50,)], [F32, F32], device, 12)).conj()
    grads = [z.imag, torch.ones(3, device=device)]
    assert grads[0].is_neg()
    before, want = [g.clone() for g in grads], _norm(grads)
    out = [torch.empty(50, device=device), torch.empty(3, device=device)]
    _check_total(clip_gradients(grads, 0.5, out=out), want)
    _check_scaled(out, before, 0.5 / (want + 1e-6))
    clip_gradients(grads, 0.5)
    _check_scaled(grads, before, 0.5 / (want + 1e-6))


def test_parameters(device):
    a, b, c = (torch.nn.Parameter(t) for t in _grads([(30,), (4, 5), (2,)], [F32] * 3, device, 9))
    a.grad, b.grad = _grads([(30,), (4, 5)], [F32] * 2, device, 10)
    before = [a.grad.clone(), b.grad.clone()]
    want = _norm(before)
    _check_total(clip_grad_norm_([a, b, c, a], 1.0), want)
    _check_scaled([a.grad, b.grad], before, 1.0 / (want + 1e-6))
    assert float(clip_grad_norm_([c], 1.0)) == 0
    one = torch.nn.Parameter(torch.zeros(3, device=device))
    one.grad = torch.ones(3, device=device)
    _check_total(clip_grad_norm_(one, None), math.sqrt(3.0))


def test_graph(device):
    grads = _grads([(1000,), (20, 20), (70_000,)], [BF16, F32, BF16], device, 11)
    out = [torch.empty_like(g, dtype=F32) for g in grads]
    for _ in range(3):
        clip_gradients(grads, 1.0, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        total = clip_gradients(grads, 1.0, out=out)
    for seed in range(3):
        for g, n in zip(grads, _grads([(1000,), (20, 20), (70_000,)], [BF16, F32, BF16], device, 20 + seed)):
            g.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        again = [torch.empty_like(o) for o in out]
        assert torch.equal(clip_gradients(grads, 1.0, out=again), total)
        assert all(torch.equal(a, b) for a, b in zip(out, again))


def test_refusals(device):
    g = torch.ones(64, device=device)
    for call, text in ((lambda: clip_gradients([g.cpu()], 1.0), "must be a CUDA tensor"), (lambda: clip_gradients([g.int()], 1.0), "not implemented"),
                       (lambda: clip_gradients([g], -1.0), "max_norm"), (lambda: clip_gradients([g], math.nan), "max_norm"),
                       (lambda: clip_gradients([g], 1.0, eps=-1.0), "eps"), (lambda: clip_gradients([g], 1.0, grad_scale=math.inf), "grad_scale"),
                       (lambda: clip_gradients([g], 1.0, out=[]), "as many"), (lambda: clip_gradients([g], 1.0, out=[g[:5]]), "shape"),
                       (lambda: clip_gradients([g, g[3:9]], 1.0), "overlaps"), (lambda: clip_gradients([g, g], 1.0), "overlaps"),
                       (lambda: clip_gradients([g, g.clone()], 1.0, out=[torch.empty(64, device=device), g]), "overlaps"),
                       (lambda: clip_gradients([g[:32]], 1.0, out=[g[16:48]]), "overlaps"),
                       (lambda: clip_gradients([g.to_sparse()], 1.0), "dense")):
        with pytest.raises(RuntimeError, match=text):
            call()
    assert (g == 1).all()
    clip_gradients([g, g], math.inf)  # only read
    clip_gradients([g, g], 1.0, out=[g.clone(), g.clone()])
    assert float(clip_gradients([], 1.0)) == 0
