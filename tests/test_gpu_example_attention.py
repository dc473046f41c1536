"""GPU tests of examples/image_transformer.py with windows, registers, causal blocks and dropout: its operators one behind the other."""
import os
import sys

import pytest
import torch
import torch.nn.functional as F

from gnnhwc import dropout
from tests.left_alone import generators_left_alone  # noqa: F401 (a fixture)
from tests import window_refs as ref

pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
try:
    import image_transformer as example
finally:
    sys.path.pop(0)

# A float32 result is off by a few units of 2^-24 of its row's size for each of some 40 products, norms and sums in a row (their
# terms' errors are independent), say 8 * 40 = 2^8.3; four times that in the norm of all.
FLOAT32 = 2.0 ** -13
# The same in bfloat16, where 12 roundings a block add in squares: sqrt(24) * 2^-8 / sqrt(3) = 2^-6.5; four times that.
BFLOAT16 = 2.0 ** -4.5


def distance(a, b):
    a, b = a.detach().double(), b.detach().double()
    return float((a - b).norm() / b.norm())


@pytest.mark.parametrize("options", [dict(window=20, registers=4), dict(causal=True, dropout=0.1), dict(window=5, registers=1, causal=True, dropout=0.3)])
def test_training_and_serving_run(options, device):
    model, losses, norms = example.train(steps=3, size=16, channels=128, blocks=2, images=2, device=device, **options)
    assert all(0 < n < float("inf") for n in losses + norms)
    for name, p in model.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all() and p.grad.any(), name
    assert example.compare_served(model, size=16, device=device) < float("inf")
    if options.get("causal"):
        assert example.compare_parts(model, 5, size=16, device=device) < BFLOAT16


@pytest.mark.parametrize("parts", [2, 7, 68])
@pytest.mark.parametrize("window,registers", [(None, 0), (13, 4)])
def test_tokens_in_parts_are_as_all_at_once(parts, window, registers, device):
    """Prompts, small parts and single tokens, against caches, in float32."""
    torch.manual_seed(1)
    model = example.ImageTransformer(128, 2, window=window, registers=registers, causal=True).to(device)
    assert example.distance_of(model, 16, 2, device, parts=parts) < FLOAT32


def plain_block(block, h, residual, positions, drops):
    """Block.forward from its formulas, in float64."""
    def norm(x, n):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + n.eps) * n.weight

    def turn(x, weight):
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + block.rotary.eps) * weight
        angles = torch.cat([positions[:, i:i + 1].double() * f.double() for i, f in enumerate(block.rotary.frequencies.split(example.HEAD // 4))], dim=1)
        c, s = angles.cos()[:, None], angles.sin()[:, None]
        even, odd = x[..., 0::2], x[..., 1::2]
        return torch.stack([even * c - odd * s, even * s + odd * c], dim=-1).flatten(-2)

    residual = residual + h
    q, k, v = F.linear(norm(residual, block.norm1), block.qkv.weight).unflatten(-1, (-1, example.HEAD)).split([block.heads, block.kv_heads, block.kv_heads], dim=2)
    q, k = turn(q, block.rotary.q_weight), turn(k, block.rotary.k_weight)
    B, L, H, D = q.shape
    k, v = (t.repeat_interleave(H // block.kv_heads, dim=2) for t in (k, v))
    seen = ref.sees(B, L, L, block.window, block.sinks, block.causal, None, False, q.device)
    scores = torch.matmul(q.transpose(1, 2), k.transpose(1, 2).transpose(2, 3)) * D ** -0.5
    mixed = torch.matmul(scores.masked_fill(~seen[:, None], -float("inf")).softmax(-1), v.transpose(1, 2)).transpose(1, 2).flatten(2)
    residual = residual + F.linear(mixed, block.out.weight) * drops[0]
    y = F.linear(F.silu(F.linear(norm(residual, block.norm2), block.up.weight)), block.down.weight)
    return y * drops[1], residual


@pytest.mark.parametrize("p", [0.0, 0.25])
def test_a_block_and_its_gradients_against_formulas(p, device):
    """All operators of a block in a row, forward and backward, in float32 against float64."""
    torch.manual_seed(2)
    block = example.Block(128, 2, window=9, sinks=2, causal=False, dropout=p).to(device)
    g = torch.Generator(device=device).manual_seed(3)
    h, residual, dy, dr = (torch.randn((2, 36, 128), generator=g, device=device) for _ in range(4))
    positions = torch.stack([torch.arange(36) // 6, torch.arange(36) % 6], dim=1).to(device)
    h.requires_grad_(True)
    weights = list(block.parameters())
    torch.manual_seed(4)
    y, r = block(h, residual, positions)
    grads = torch.autograd.grad([y, r], [h, *weights], [dy, dr])
    torch.manual_seed(4)
    ones = torch.ones_like(h)
    drops = [dropout(ones, p, int(torch.empty((), dtype=torch.int64).random_())).detach().double() if p else 1.0 for _ in range(2)]
    wide = example.Block(128, 2, window=9, sinks=2, causal=False, dropout=p).to(device).double()
    wide.load_state_dict({n: t.double() for n, t in block.state_dict().items()})
    h64 = h.detach().double().requires_grad_(True)
    y64, r64 = plain_block(wide, h64, residual.double(), positions, drops)
    want = torch.autograd.grad([y64, r64], [h64, *wide.parameters()], [dy.double(), dr.double()])
    for name, a, b in zip(["y", "residual", "h"] + [n for n, _ in block.named_parameters()], [y, r, *grads], [y64, r64, *want]):
        assert distance(a, b) < FLOAT32, (name, distance(a, b))


@pytest.mark.parametrize("options", [dict(window=20, registers=4), dict(causal=True, dropout=0.1), dict(window=5, registers=1, causal=True, dropout=0.3)])
def test_the_8_bit_form_stays_near_the_other(options, device):
    """e4m3 values are off by 2.6 % in the mean; a block's products average over channels, and the residual stream is not quantised."""
    model, _losses, _norms = example.train(steps=3, size=16, channels=128, blocks=2, images=2, device=device, **options)
    assert example.compare_served(model, size=16, device=device) < 0.05
