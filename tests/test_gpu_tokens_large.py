"""GPU tests of the operators for token streams at offsets beyond 32 bits and at more threads than one launch has."""
import pytest
import torch

from gnnhwc import clip_gradients, rms_norm, rms_norm_quant, rotary, rotary_frequencies

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _free():
    torch.cuda.empty_cache()


def test_rows_far_apart(device):
    """Rows 3 GiB of elements apart, and what follows the 32-bit limits in bytes and in elements."""
    C, stride = 200, 3 << 30
    big = torch.empty(2 * stride + C, dtype=BF16, device=device)
    x = big.as_strided((3, C), (stride, 1))
    values = torch.randn(3, C, device=device).to(BF16)
    x.copy_(values)
    w = torch.randn(C, device=device)
    want = rms_norm(values, w, residual=values, return_sum=True)
    got = rms_norm(x, w, residual=x, return_sum=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(rms_norm_quant(x, w)[0].view(torch.uint8), rms_norm_quant(values, w)[0].view(torch.uint8))
    a, b = x.detach().requires_grad_(True), values.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(rms_norm(a, w), a, values)[0], torch.autograd.grad(rms_norm(b, w), b, values)[0])
    f, p = rotary_frequencies((48,), device=device), torch.arange(3, device=device)
    assert torch.equal(rotary(x.view(1, 3, 1, C), None, p, f), rotary(values.view(1, 3, 1, C), None, p, f))
    assert torch.equal(rotary(x.view(3, 1, 1, C), None, p.view(3, 1), f), rotary(values.view(3, 1, 1, C), None, p.view(3, 1), f))
    del big, x, a
    _free()


def test_more_elements_than_32_bits(device):
    rows, C = (1 << 32) // 1024 + 3, 1024  # 8.6 GB
    x = torch.empty((rows, C), dtype=BF16, device=device).normal_()
    y = rms_norm(x)
    for i in (0, 12345, (1 << 31) // C, rows - 1):
        assert torch.equal(y[i], rms_norm(x[i:i + 1])[0]), i
    del y
    total = clip_gradients([x], float("inf"))
    want = sum(float(p.double().square().sum()) for p in x.split(1 << 18)) ** 0.5
    assert abs(float(total) - want) <= 4 * 2.0 ** -24 * want
    last = x[-1].clone()
    total = clip_gradients([x], 1.0)
    factor = 1.0 / (want + 1e-6)
    assert torch.allclose(x[-1].float(), last.float() * factor, rtol=2.0 ** -8, atol=0)
    del x
    _free()


def test_more_threads_than_a_launch(device):
    rows = (1 << 29) + 5  # of one lane vector each, eight lanes a row
    x = torch.empty((rows, 8), dtype=BF16, device=device).normal_()
    y, s = rms_norm(x, residual=x, return_sum=True)
    q, scales = rms_norm_quant(x)
    for at in (0, (1 << 28) - 2, (1 << 29) - 2, rows - 4):
        part = x[at:at + 4]
        a, b = rms_norm(part, residual=part, return_sum=True)
        assert torch.equal(y[at:at + 4], a) and torch.equal(s[at:at + 4], b), at
        c, d = rms_norm_quant(part)
        assert torch.equal(q[at:at + 4].view(torch.uint8), c.view(torch.uint8)) and torch.equal(scales[at:at + 4], d), at
    del x, y, s, q, scales
    _free()


def test_many_tokens_of_one_head(device):
    tokens = (1 << 28) + 7
    q = torch.empty((1, tokens, 1, 8), dtype=BF16, device=device).normal_()
    p = torch.arange(tokens, device=device, dtype=torch.int32) & 0xffff
    f = rotary_frequencies((4,), device=device)
    y = rotary(q, None, p, f)
    for at in (0, 1 << 27, tokens - 5):
        assert torch.equal(y[:, at:at + 5], rotary(q[:, at:at + 5], None, p[at:at + 5], f)), at
    del q, y, p
    _free()
