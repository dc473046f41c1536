"""GPU test of the 8-bit norms' last step: q is the float32 quotient y / scale, rounded to nearest even.  Rows of +-1 have a norm of
one, so that y is the weight; the weights are chosen where a quotient lies on the middle between two 8-bit values or next to it,
so that one rounding more, as of y * (1 / scale), is seen."""
import pytest
import torch

from gnnhwc import rms_norm_quant

pytestmark = pytest.mark.gpu
MOST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def _middles(out, shape, g):
    """Values halfway between two neighbours of the type."""
    if out == torch.int8:
        return torch.randint(-126, 126, shape, generator=g).float() + 0.5
    exponent = torch.randint(-5, 9, shape, generator=g).float()
    m = (8 + torch.randint(0, 8, shape, generator=g).float() + 0.5) / 8 * 2.0 ** exponent
    m = torch.where(m < 448.0, m, m / 16)
    return torch.where(torch.rand(shape, generator=g) < 0.5, m, -m)


@pytest.mark.parametrize("out", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("C,block", [(16384, 16), (4096, 64), (2560, 256), (1008, 16)])
def test_quotients_at_the_middles(C, block, out, device):
    g = torch.Generator().manual_seed(C + block)
    n = -(-C // block)
    most = torch.exp(4 * torch.randn(n, 1, generator=g)).float()
    scale = most / MOST[out]
    w = _middles(out, (n, block), g) * scale
    # the product's neighbours, too
    step = torch.randint(-1, 2, w.shape, generator=g, dtype=torch.int32)
    w = (w.view(torch.int32) + step).view(torch.float32)
    w = torch.where(w.abs() < most, w, most / 3)
    w[:, 0:1] = most  # the largest of its block
    w = w.reshape(-1)[:C]
    x = torch.where(torch.rand(3, C, generator=g) < 0.5, -1.0, 1.0)
    q, scales = rms_norm_quant(x.to(device), w.to(device), 0.0, out_dtype=out, block=block)
    assert torch.equal(scales.cpu(), scale.view(1, n).expand(3, n))
    y = x * w
    units = torch.cat([p / scale[i] for i, p in enumerate(y.split(block, dim=1))], dim=1)
    want = units.round() if out == torch.int8 else units.to(out).float()
    assert torch.equal(q.cpu().float(), want), int((q.cpu().float() != want).sum())


def test_quotients_of_rows(device):
    """One scale a row: the weights' middles lie at the scale that all rows share."""
    g = torch.Generator().manual_seed(5)
    for out in MOST:
        for C in (72, 1111, 5120):
            most = torch.tensor([[2.7182817]])
            scale = most / MOST[out]
            w = (_middles(out, (1, C), g) * scale).clamp(-2.7, 2.7)
            w[0, C // 2] = most
            x = torch.where(torch.rand(5, C, generator=g) < 0.5, -1.0, 1.0)
            q, scales = rms_norm_quant(x.to(device), w[0].to(device), 0.0, out_dtype=out)
            assert torch.equal(scales.cpu(), scale.expand(5, 1))
            units = x * w / scale
            want = units.round() if out == torch.int8 else units.to(out).float()
            assert torch.equal(q.cpu().float(), want)


def test_infinite_weights(device):
    """A scale that is infinite leaves zeros beside the infinity, as the quotient does."""
    w = torch.linspace(-3, 3, 64)
    w[5] = float("inf")
    for out in MOST:
        q, scales = rms_norm_quant(torch.ones(2, 64, device=device), w.to(device), 0.0, out_dtype=out, block=32)
        assert (scales[:, 0] == float("inf")).all() and scales[:, 1].isfinite().all()
        values = q.float()[:, :32]
        others = torch.arange(32, device=device) != 5
        assert (values[:, others] == 0).all()
        assert values[:, 5].isnan().all() if out == torch.float8_e4m3fn else (values[:, 5] == 0).all()
