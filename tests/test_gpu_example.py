"""GPU test of examples/image_transformer.py: the operators together, in training and in serving."""
import os
import sys

import pytest

pytestmark = pytest.mark.gpu
EXAMPLES = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples")


def test_the_image_transformer_learns_and_serves(device):
    sys.path.insert(0, EXAMPLES)
    try:
        import image_transformer as example
    finally:
        sys.path.remove(EXAMPLES)
    model, losses, norms = example.train(steps=25, size=24, channels=128, blocks=2, images=4, device=device)
    assert losses[-1] < 0.7 * losses[0] and all(n > 0 and n < float("inf") for n in norms), (losses[0], losses[-1])
    # e4m3 values are off by 2.6 % in the mean; a block's products average over channels, and the residual stream is not quantised
    assert example.compare_served(model, size=24, device=device) < 0.05
