"""A fixture for tests that seed torch's generators: what runs behind them draws what it would have drawn without them."""
import pytest
import torch


@pytest.fixture(autouse=True)
def generators_left_alone():
    states = torch.get_rng_state(), torch.cuda.get_rng_state_all()
    yield
    torch.set_rng_state(states[0])
    torch.cuda.set_rng_state_all(states[1])
