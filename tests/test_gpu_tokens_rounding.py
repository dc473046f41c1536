"""GPU test of how often a float32 norm rounds: rows of one repeated value, whose norm is 1.

The mean square of a relative rounding error of float32 values spread over a binade is (2 u)^2 / 12 / 2 (u = 2^-24; an error is
uniform within half a unit in the last place, and 1 / m^2 is 1/2 on average over [1, 2)), i.e. (0.408 u)^2.  A result takes three
of them, each on its own: the division of the sum by C (halved by the root), 1 / sqrt, and the product.  The sum of squares takes
one for each of up to `chain` steps, halved as well.  Anything beyond is a rounding that the formula does not need."""
import math

import pytest
import torch

from gnnhwc import rms_norm

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.mark.parametrize("C,chain", [(3, 3), (7, 5), (15, 6), (100, 9)])
def test_rows_of_one_value(C, chain, device):
    g = torch.Generator(device=device).manual_seed(C)
    t = 1 + torch.rand((500_000, 1), dtype=torch.float64, generator=g, device=device)
    t = t * torch.where(torch.rand(t.shape, generator=g, device=device) < 0.5, 1.0, 2 ** 0.5)  # both kinds of exponent for the root
    y = rms_norm(t.float().expand(-1, C), None, 0.0).double()
    error = float((y - 1).square().mean().sqrt())
    allowed = 0.408 * U * math.sqrt(chain / 4 + 1 / 4 + 1 + 1)
    print("rows of %d: %.3f u, allowed %.3f u" % (C, error / U, allowed / U), flush=True)
    assert error <= allowed
