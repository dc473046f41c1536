"""GPU test of clip_grad_norm_ called as torch.nn.utils.clip_grad_norm_ is."""
import math

import pytest
import torch

from gnnhwc import clip_grad_norm_

pytestmark = pytest.mark.gpu


def test_torchs_call(device):
    """The third argument is torch.nn.utils.clip_grad_norm_'s: which norm."""
    def parameters():
        g = torch.Generator().manual_seed(1)
        ps = [torch.nn.Parameter(torch.zeros(30, 7, device=device)), torch.nn.Parameter(torch.zeros(11, device=device))]
        for p in ps:
            p.grad = torch.randn(p.shape, generator=g).to(device)
        return ps

    ours, theirs = parameters(), parameters()
    a, b = clip_grad_norm_(ours, 1.0, 2.0), torch.nn.utils.clip_grad_norm_(theirs, 1.0, 2.0)
    assert math.isclose(float(a), float(b), rel_tol=1e-6)
    for p, q in zip(ours, theirs):
        assert torch.allclose(p.grad, q.grad, rtol=1e-6, atol=0)
    before = [p.grad.clone() for p in ours]
    for kind in (1.0, math.inf, 1 / 1024):
        with pytest.raises(RuntimeError, match="norm_type"):
            clip_grad_norm_(ours, 1.0, kind)
    with pytest.raises(TypeError):
        clip_grad_norm_(ours, 1.0, 2.0, 0.5)
    assert all(torch.equal(p.grad, g) for p, g in zip(ours, before))
    ours, theirs = parameters(), parameters()
    total = clip_grad_norm_(ours, 1.0, grad_scale=0.5)
    for p in theirs:
        p.grad.mul_(0.5)
    want = torch.nn.utils.clip_grad_norm_(theirs, 1.0, norm_type=2)
    assert math.isclose(float(total), float(want), rel_tol=1e-6)
    for p, q in zip(ours, theirs):
        assert torch.allclose(p.grad, q.grad, rtol=1e-6, atol=0)
