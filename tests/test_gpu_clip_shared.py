"""GPU tests of what clip_gradients does with tensors whose elements share memory, and of what it writes when it only has to look."""
import math

import pytest
import torch

from gnnhwc import clip_gradients

pytestmark = pytest.mark.gpu


def test_elements_that_share_memory(device):
    """A gradient that is one value for all, as that of a sum: its norm can be had, but it cannot be written."""
    one = torch.full((1,), 0.5, device=device)
    other = torch.ones(16, device=device)
    shared = one.expand(16)
    total = clip_gradients([other, shared], math.inf)
    assert math.isclose(float(total), math.sqrt(16 + 16 * 0.25), rel_tol=1e-6)
    version = other._version
    for call in (lambda: clip_gradients([other, shared], 1.0), lambda: clip_gradients([other], 1.0, out=[shared]),
                 lambda: clip_gradients([other, shared], math.inf, grad_scale=0.5)):
        with pytest.raises(RuntimeError, match="share memory"):
            call()
        assert (other == 1).all() and float(one) == 0.5 and other._version == version  # refused before anything is written
    out = [torch.empty(16, device=device) for _ in range(2)]
    clip_gradients([other, shared], 1.0, out=out)
    assert torch.allclose(out[1], torch.full_like(other, 0.5 / (float(total) + 1e-6)), rtol=1e-6)


def test_the_norm_alone_writes_nothing(device):
    """Not into a strided gradient either, which another computation may be about to read on its own terms."""
    wide = torch.arange(24, device=device, dtype=torch.float32).view(4, 6)
    strided = wide[:, ::2]
    version = wide._version
    total = clip_gradients([strided], math.inf)
    assert math.isclose(float(total), float(strided.norm()), rel_tol=1e-6) and wide._version == version
