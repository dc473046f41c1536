"""CPU checks of what the compiler made of the attention kernels: no register lies in scratch memory (wavefronts count the copies that
they wait for, and an access to scratch memory would be among them), and as many workgroups fit a CU as they are bound for."""
import re

import pytest

from gnnhwc import _cabi
from tests.test_kernel_resources import LDS_PER_CU, _kernels


@pytest.fixture(scope="module")
def kernels():
    assert _cabi.lib is not None
    return {n: k for n, k in _kernels().items() if re.search(r"\d+(window|dropout)_\w*kernel", n)}


def test_no_scratch(kernels):
    seen = {re.search(r"\d+(window_\w+?|dropout)_kernel", n).group(1) for n in kernels}
    assert seen == {"window_forward", "window_few", "window_join", "window_dq", "window_dq_sum", "window_dkv", "window_sink", "window_sum", "dropout"}
    for name, k in kernels.items():
        assert k[".vgpr_spill_count"] == 0 and k[".private_segment_fixed_size"] == 0, name


def test_shared_memory_fits(kernels):
    for name, k in kernels.items():
        assert k[".group_segment_fixed_size"] <= LDS_PER_CU, name
