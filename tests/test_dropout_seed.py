"""Where Dropout's seeds come from: torch's CPU generator, whatever torch's default device is."""
import sys

import pytest
import torch

from gnnhwc import Dropout
from tests.left_alone import generators_left_alone  # noqa: F401 (a fixture)


def seeds(monkeypatch, **where):
    """The seeds that three calls on a host tensor would hand to the kernel."""
    got = []
    monkeypatch.setattr(sys.modules["gnnhwc.dropout"], "dropout", lambda x, p, seed, *rest: got.append(seed))
    m, x = Dropout(0.5), torch.ones(3, device="cpu")
    torch.manual_seed(4)
    for _ in range(3):
        if where:
            with torch.device(where["device"]):
                m(x)
        else:
            m(x)
    return got


def test_the_default_device_has_no_say(monkeypatch):
    plain = seeds(monkeypatch)
    assert len(set(plain)) == 3 and all(type(s) is int for s in plain)
    assert seeds(monkeypatch, device="meta") == plain


@pytest.mark.gpu
def test_masks_are_the_same_under_a_default_device(device):
    m, x = Dropout(0.5), torch.ones(4096, device=device)
    torch.manual_seed(4)
    want = [m(x) for _ in range(2)]
    torch.manual_seed(4)
    with torch.device(device):
        got = [m(x) for _ in range(2)]
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and not torch.equal(*want)
