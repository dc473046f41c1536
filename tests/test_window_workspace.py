"""CPU checks that the header says of the attention's workspace what its functions hold a caller to."""
import ctypes
import os
import re

import pytest

from gnnhwc import _cabi
from tests.test_attention_cpu import _block, _call

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "gnnhwc_tokens.h")
lib = _cabi.lib


def _alignment():
    return int(re.search(r"#define GNNHWC_WINDOW_WORKSPACE_ALIGNMENT \(\(size_t\)(\d+)\)", open(HEADER).read()).group(1))


def test_the_conventions_except_it():
    """The alignment that is enough for all others is named with its exception."""
    sentence, = re.findall(r"\(8-byte aligned is enough[^)]*\)", open(HEADER).read().replace("\n * ", " "))
    assert "GNNHWC_WINDOW_WORKSPACE_ALIGNMENT" in sentence


@pytest.mark.parametrize("backward", [False, True])
def test_addresses(backward):
    """Half of it is refused, and what is enough for the other functions, by a call that needs a workspace."""
    run = lib.gnnhwc_window_bwd if backward else lib.gnnhwc_window
    c, _keep = _call(batch=1, keys=5000, window=-1)  # several workgroups share a head's keys
    _raw, ws = _block()
    ws -= ws % _alignment()
    assert run(ctypes.byref(c), ws + _alignment() // 2, 1 << 40, None) == -2 and "misaligned" in _cabi.last_error()
    assert run(ctypes.byref(c), ws + 8, 1 << 40, None) == -2  # (what the others take)


def test_a_backward_of_nothing_takes_an_aligned_one():
    c, _keep = _call(batch=0)
    _raw, ws = _block()
    ws += -ws % _alignment()
    for n in range(3):
        assert lib.gnnhwc_window_bwd(ctypes.byref(c), ws + n * _alignment(), 1 << 20, None) == 0
        assert lib.gnnhwc_window_bwd(ctypes.byref(c), ws + n * _alignment() + _alignment() // 2, 1 << 20, None) == -2
