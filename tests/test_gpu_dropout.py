"""GPU tests of dropout against its definition, the words computed with numpy's integers."""
import math

import numpy as np
import pytest
import torch

from gnnhwc import Dropout, dropout
from tests.dropout_refs import bits_of
from tests.left_alone import generators_left_alone  # noqa: F401 (a fixture)
from tests.token_refs import LEAST, U

pytestmark = pytest.mark.gpu
F32, F64, F16, BF16 = torch.float32, torch.float64, torch.float16, torch.bfloat16


def normal(shape, dtype, device, seed):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return torch.randn(shape, generator=g, dtype=F64).to(dtype).to(device)


def masked(x, p, seed, offset, residual=None):
    """(value in float64, truth values of what is kept)."""
    least = math.floor(p * 65536 + 0.5)
    keep = torch.from_numpy(bits_of(x.numel(), seed, offset) >= least).to(x.device).view(x.shape)
    y = torch.where(keep, x.double() * (65536 / (65536 - least) if least < 65536 else 0.0), 0.0)
    return (y if residual is None else y + residual.double()), keep


def check(got, want, terms):
    """One rounding to the type; before it the scale, the product and the sum are rounded in float32 (float64): three half units of
    the terms' magnitude."""
    compute = 2.0 ** -53 if got.dtype == F64 else 2.0 ** -24
    assert ((got.double() - want).abs() <= U[got.dtype] * want.abs() + LEAST[got.dtype] + 4 * compute * terms).all()


# sizes around a counter's 8 elements, a lane's and a workgroup's share; the last ones whole workgroups and a rest
@pytest.mark.parametrize("dtype", [F32, F64, F16, BF16])
@pytest.mark.parametrize("n", [1, 7, 8, 9, 63, 2047, 2048, 2049, 4096, 8191, 8192, 8193, 100003, 65536])
def test_forward_and_backward(n, dtype, device):
    for i, (p, residual) in enumerate(((0.1, False), (0.5, True), (0.9, False), (0.25, True))):
        print("dropout", n, dtype, p, residual, flush=True)
        x = normal((n,), dtype, device, i).requires_grad_(True)
        r = normal((n,), dtype, device, 10 + i).requires_grad_(True) if residual else None
        dy = normal((n,), dtype, device, 20 + i)
        y = dropout(x, p, 1234 + i, 7 * i, residual=r)
        want, keep = masked(x.detach(), p, 1234 + i, 7 * i, None if r is None else r.detach())
        check(y.detach(), want, x.detach().double().abs() / (1 - p) + (0 if r is None else r.detach().double().abs()))
        got = torch.autograd.grad(y, [x] if r is None else [x, r], dy)
        want, _ = masked(dy, p, 1234 + i, 7 * i)
        check(got[0], want, want.abs())
        assert not got[0][~keep].any()
        if r is not None:
            assert torch.equal(got[1], dy)


def test_extremes_of_p(device):
    x = normal((5000,), F32, device, 1)
    r = normal((5000,), F32, device, 2)
    assert torch.equal(dropout(x, 0.0, 3), x) and torch.equal(dropout(x, 0, 3, residual=r), x + r)
    assert not dropout(x, 1.0, 3).any() and torch.equal(dropout(x, 1, 3, residual=r), r)
    assert torch.equal(dropout(x, 2.0 ** -18, 3), x)  # less than half of 2^-16
    least = dropout(torch.ones(1 << 20, device=device), 1.0 - 2.0 ** -16, 3)
    assert set(least.unique().tolist()) == {0.0, 65536.0}


def test_what_is_dropped_has_no_effect(device):
    for dtype in (F32, F16, BF16):
        x = torch.full((4096,), math.nan, dtype=dtype, device=device)
        x[::2] = math.inf
        _, keep = masked(x.float(), 0.5, 11, 0)
        y = dropout(x, 0.5, 11)
        assert not y[~keep].any() and not torch.isfinite(y[keep]).any()
        r = normal((4096,), dtype, device, 1)
        assert torch.equal(dropout(x, 0.5, 11, residual=r)[~keep], r[~keep])


def test_seeds_and_offsets(device):
    """64 bits of each count; integers of any sign; a tensor gives what its integer gives."""
    x = torch.ones(4096, device=device)
    seen = []
    for seed, offset in ((0, 0), (1, 0), (0, 1), (2 ** 32, 0), (0, 2 ** 32), (2 ** 63 + 5, 2 ** 63 + 9), (-1, -1), (2 ** 64 - 1, 0)):
        y = dropout(x, 0.5, seed, offset)
        assert torch.equal(y.double(), masked(x, 0.5, seed % 2 ** 64, offset % 2 ** 64)[0]), (seed, offset)
        at = torch.tensor(seed - 2 ** 64 if seed >= 2 ** 63 else seed, device=device)
        assert torch.equal(dropout(x, 0.5, at, offset), y)
        assert torch.equal(dropout(x, 0.5, at.view(1), offset), y)
        seen.append(y)
    assert all(not torch.equal(a, b) for i, a in enumerate(seen) for b in seen[:i])


def test_share_of_dropped(device):
    """2^22 elements: the share's deviation is sqrt(p (1 - p) / n), held to six of them; neighbours are as independent."""
    n = 1 << 22
    for p in (0.05, 0.1, 0.5):
        keep = dropout(torch.ones(n, device=device), p, 99) > 0
        q = 1 - math.floor(p * 65536 + 0.5) / 65536
        assert abs(float(keep.double().mean()) - q) < 6 * math.sqrt(q * (1 - q) / n)
        both = (keep[1:] & keep[:-1]).double().mean()
        assert abs(float(both) - q * q) < 6 * math.sqrt(3 / n) * q


def test_layouts_and_places(device):
    """An element's place decides, not its memory."""
    x = normal((6, 5, 40), BF16, device, 1)
    y = dropout(x, 0.3, 5)
    assert torch.equal(dropout(x.transpose(0, 1).contiguous().transpose(0, 1), 0.3, 5), y)
    assert torch.equal(dropout(torch.cat([x, x], -1)[..., :40], 0.3, 5), y)
    flat = torch.zeros(x.numel() + 3, dtype=BF16, device=device)
    flat[3:] = x.flatten()
    assert torch.equal(dropout(flat[3:].view(x.shape), 0.3, 5), y)
    image = normal((2, 24, 7, 5), BF16, device, 2).to(memory_format=torch.channels_last)
    z = dropout(image, 0.3, 6, channel_dim=1)
    assert z.shape == image.shape and z.stride(1) == 1
    assert torch.equal(z.permute(0, 2, 3, 1), dropout(image.permute(0, 2, 3, 1).contiguous(), 0.3, 6))
    # the gradient of a sum is expanded from one value
    x = x.clone().requires_grad_(True)
    g, = torch.autograd.grad(dropout(x, 0.3, 5).sum(), x)
    assert torch.equal(g, dropout(torch.ones_like(g), 0.3, 5))


def test_derivatives(device):
    x, r = normal((300,), F64, device, 1).requires_grad_(True), normal((300,), F64, device, 2).requires_grad_(True)
    assert torch.autograd.gradcheck(lambda a, b: dropout(a, 0.4, 3, residual=b), (x, r))
    assert torch.autograd.gradgradcheck(lambda a, b: dropout(a, 0.4, 3, residual=b), (x, r))


def test_module(device):
    m = Dropout(0.2)
    x, r = normal((64, 80), F32, device, 1), normal((64, 80), F32, device, 2)
    torch.manual_seed(4)
    a, b = m(x), m(x)
    torch.manual_seed(4)
    assert torch.equal(m(x), a) and not torch.equal(a, b)
    assert (m(x, r) == r).any() and torch.equal(m.eval()(x), x) and torch.equal(m(x, r), x + r)
    # a recomputed forward draws the same seed
    leaf = x.clone().requires_grad_(True)
    m.train()
    y = torch.utils.checkpoint.checkpoint(lambda t: m(t), leaf, use_reentrant=False)
    g, = torch.autograd.grad(y, leaf, torch.ones_like(y))
    assert torch.equal(g != 0, y.detach() != 0)


def test_captured(device):
    """A seed tensor is read at each replay; forward and backward see the same one."""
    x = normal((1000, 80), BF16, device, 1).requires_grad_(True)
    dy = normal((1000, 80), BF16, device, 2)
    seed = torch.tensor(1, device=device)

    def step():
        y = dropout(x, 0.5, seed, 3)
        return y, torch.autograd.grad(y, x, dy)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, g = step()
    for s in (5, 6, 7):
        seed.fill_(s)
        graph.replay()
        torch.cuda.synchronize()
        with torch.no_grad():
            assert torch.equal(y, dropout(x, 0.5, s, 3)) and torch.equal(g, dropout(dy, 0.5, s, 3))


def test_operator(device):
    x, r = normal((33, 8), F32, device, 1).requires_grad_(True), normal((33, 8), F32, device, 2).requires_grad_(True)
    torch.library.opcheck(torch.ops.gnop.dropout, (x, r, 0.3, 5, None, 0))
    compiled = torch.compile(lambda a, b: dropout(a, 0.3, 5, residual=b), fullgraph=True, backend="aot_eager")
    assert torch.equal(compiled(x, r), dropout(x, 0.3, 5, residual=r))


def test_more_than_32_bits_of_elements(device):
    """Places beyond 2^32: the counter's upper word."""
    n = (1 << 32) + 16 * 8
    x = torch.ones(n, dtype=BF16, device=device)
    y = dropout(x, 0.5, 77)
    for at in (0, (1 << 32) - 64, 1 << 32):
        keep = bits_of(64, 77, 0, first=at) >= 32768
        assert np.array_equal((y[at:at + 64] > 0).cpu().numpy(), keep)


def test_refusals(device):
    x = normal((4, 8), F32, device, 1)
    for call, text in ((lambda: dropout(x, -0.1, 1), "p must"), (lambda: dropout(x, 1.5, 1), "p must"), (lambda: dropout(x, math.nan, 1), "p must"),
                       (lambda: dropout(x, 0.5, 1, residual=x[:2]), "residual"), (lambda: dropout(x, 0.5, 1, residual=x.half()), "residual"),
                       (lambda: dropout(x, 0.5, torch.tensor([1, 2], device=device)), "seed"), (lambda: dropout(x, 0.5, torch.tensor(1)), "CUDA"),
                       (lambda: dropout(x.int(), 0.5, 1), "not implemented")):
        with pytest.raises(RuntimeError, match=text):
            call()
