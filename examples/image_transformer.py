"""A small image transformer on the framework's operators: GroupNorm over channels-last features (GN_NHWC), then transformer
blocks over the pixels as tokens (RMSNorm with the residual's addition, Rotary with two axes and normalised heads), trained in
bfloat16 with float32 master weights (clip_gradients writes the clipped float32 gradients), and served with 8-bit norms
(rms_norm_quant).  Needs a GPU:

  python examples/image_transformer.py [--steps 30] [--size 32] [--channels 256] [--blocks 2]

It learns to undo noise on synthetic images and prints the loss, the gradient norm and how far the 8-bit form is from the other.
"""
import argparse
import os
import sys

import torch
import torch.nn as nn
import torch.nn.functional as F

_PACKAGES = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "channels-last-groupnorm_amd")
if _PACKAGES not in sys.path:
    sys.path.insert(0, _PACKAGES)

from gnnhwc import GN_NHWC, RMSNorm, Rotary, clip_gradients, rms_norm_quant  # noqa: E402

HEAD = 64
PATCH = 2


def attention(q, k, v):
    """softmax(q k^T / sqrt(D)) v in float32; q: (B, L, H, D), k, v: (B, L, K, D), H a multiple of K."""
    q, k, v = (t.float().transpose(1, 2).contiguous() for t in (q, k, v))
    k, v = (t.repeat_interleave(q.shape[1] // t.shape[1], dim=1) for t in (k, v))
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()) * q.shape[-1] ** -0.5
    return torch.matmul(scores.softmax(dim=-1), v).transpose(1, 2).flatten(2)


class Block(nn.Module):
    def __init__(self, channels, kv_heads=2):
        super().__init__()
        self.heads, self.kv_heads = channels // HEAD, kv_heads
        self.norm1, self.norm2 = RMSNorm(channels), RMSNorm(channels)
        self.qkv = nn.Linear(channels, (self.heads + 2 * kv_heads) * HEAD, bias=False)
        self.rotary = Rotary(HEAD, (HEAD // 4, HEAD // 4), interleaved=True, qk_norm=True)
        self.out = nn.Linear(channels, channels, bias=False)
        self.up, self.down = nn.Linear(channels, 4 * channels, bias=False), nn.Linear(4 * channels, channels, bias=False)

    def mix(self, qkv, positions):
        B, L, _ = qkv.shape
        q, k, v = qkv.split([self.heads * HEAD, self.kv_heads * HEAD, self.kv_heads * HEAD], dim=-1)
        q, k = self.rotary(q.unflatten(-1, (self.heads, HEAD)), k.unflatten(-1, (self.kv_heads, HEAD)), positions)
        return self.out(attention(q, k, v.unflatten(-1, (self.kv_heads, HEAD))).to(qkv.dtype))

    def forward(self, h, residual, positions):
        """h is added to the residual stream by the norm that reads both."""
        n, residual = self.norm1(h, residual)
        n, residual = self.norm2(self.mix(self.qkv(n), positions), residual)
        return self.down(F.silu(self.up(n))), residual

    def serve(self, h, residual, positions):
        """The same with both norms leaving in 8 bits, a scale per token, which is one for each row of a product and is applied
        to its result.  (The weights here stay in bfloat16, and the 8-bit values are widened in front of the product; a serving
        program hands them to an 8-bit one as they are.)"""
        def product(q, scales, linear):
            return (F.linear(q.to(linear.weight.dtype), linear.weight) * scales).to(linear.weight.dtype)

        q, scales, residual = rms_norm_quant(h, self.norm1.weight, self.norm1.eps, residual=residual, return_sum=True)
        h = self.mix(product(q, scales, self.qkv), positions)
        q, scales, residual = rms_norm_quant(h, self.norm2.weight, self.norm2.eps, residual=residual, return_sum=True)
        return self.down(F.silu(product(q, scales, self.up))), residual


class ImageTransformer(nn.Module):
    def __init__(self, channels=256, blocks=2):
        super().__init__()
        self.stem = nn.Linear(3 * PATCH * PATCH, channels)
        self.features = GN_NHWC(32, channels, activation="silu")
        self.blocks = nn.ModuleList(Block(channels) for _ in range(blocks))
        self.norm = RMSNorm(channels)
        self.head = nn.Linear(channels, 3 * PATCH * PATCH)

    def forward(self, images, eight_bits=False):
        B, _, H, W = images.shape
        h, w = H // PATCH, W // PATCH
        patches = images.unflatten(2, (h, PATCH)).unflatten(4, (w, PATCH)).permute(0, 2, 4, 1, 3, 5).flatten(3)
        x = self.stem(patches).permute(0, 3, 1, 2)  # (B, C, h, w) in channels-last memory
        residual = self.features(x).permute(0, 2, 3, 1).flatten(1, 2)  # the same memory as tokens
        grid = torch.meshgrid(torch.arange(h, device=x.device), torch.arange(w, device=x.device), indexing="ij")
        positions = torch.stack(grid, dim=-1).view(h * w, 2)
        y = torch.zeros_like(residual)
        for block in self.blocks:
            y, residual = (block.serve if eight_bits else block)(y, residual, positions)
        y, _ = self.norm(y, residual)
        out = self.head(y).view(B, h, w, 3, PATCH, PATCH)
        return out.permute(0, 3, 1, 4, 2, 5).reshape(images.shape)


def batch(n, size, generator, device):
    """(noisy, clean) images: smooth waves of random direction and phase."""
    grid = torch.linspace(0, 6.28, size, device=device)
    a = torch.rand((n, 3, 3, 1, 1), generator=generator, device=device)
    clean = torch.sin(grid.view(1, 1, size, 1) * (1 + a[:, 0]) + grid.view(1, 1, 1, size) * (1 + a[:, 1]) + 6.28 * a[:, 2])
    noise = 0.5 * torch.empty_like(clean).normal_(generator=generator)
    return (clean + noise).bfloat16(), clean.bfloat16()


def train(steps=30, size=32, channels=256, blocks=2, images=8, max_norm=1.0, device="cuda", say=lambda *a: None):
    """Returns the model, its losses and the gradient norms."""
    torch.manual_seed(0)
    model = ImageTransformer(channels, blocks).to(device).bfloat16()
    parameters = list(model.parameters())
    masters = [p.detach().float() for p in parameters]
    for m in masters:
        m.grad = torch.zeros_like(m)
    optimiser = torch.optim.AdamW(masters, lr=2e-3)
    generator = torch.Generator(device=device).manual_seed(1)
    losses, norms = [], []
    for step in range(steps):
        noisy, clean = batch(images, size, generator, device)
        loss = F.mse_loss(model(noisy).float(), clean.float())
        model.zero_grad()
        loss.backward()
        # bfloat16 gradients in, clipped float32 gradients out; nothing waits for the norm
        norms.append(clip_gradients([p.grad for p in parameters], max_norm, out=[m.grad for m in masters]))
        optimiser.step()
        with torch.no_grad():
            for p, m in zip(parameters, masters):
                p.copy_(m)
        losses.append(loss.detach())
        if step % 10 == 0 or step == steps - 1:
            say("step %3d  loss %.4f  gradient norm %.3f" % (step, float(losses[-1]), float(norms[-1])))
    return model, [float(v) for v in losses], [float(v) for v in norms]


@torch.no_grad()
def compare_served(model, size=32, images=4, device="cuda"):
    """Relative distance of the 8-bit form's result from the other's."""
    noisy, _ = batch(images, size, torch.Generator(device=device).manual_seed(2), device)
    a, b = model(noisy).float(), model(noisy, eight_bits=True).float()
    return float((a - b).norm() / a.norm())


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=30)
    ap.add_argument("--size", type=int, default=32)
    ap.add_argument("--channels", type=int, default=256)
    ap.add_argument("--blocks", type=int, default=2)
    a = ap.parse_args()
    model, losses, _ = train(a.steps, a.size, a.channels, a.blocks, say=lambda *s: print(*s, flush=True))
    print("loss %.4f -> %.4f, 8-bit norms differ by %.2f %%" % (losses[0], losses[-1], 100 * compare_served(model, a.size)))


if __name__ == "__main__":
    main()
