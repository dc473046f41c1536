"""CPU checks of what the compiler made of the token kernels: nothing of a call that fits 256 threads lies in scratch memory, and
what a walk counts on being resident together is."""
import re

import pytest

from gnnhwc import _cabi
from tests.test_kernel_resources import _kernels, _workgroups_per_cu


@pytest.fixture(scope="module")
def kernels():
    assert _cabi.lib is not None
    return {n: k for n, k in _kernels().items() if re.search(r"rms_fwd|rms_bwd|rotary_|clip_|partial_sum", n)}


def test_no_scratch(kernels):
    seen = set()
    for name, k in kernels.items():
        seen.add(re.search(r"rms_fwd|rms_bwd|rotary_norm_bwd|rotary|clip|partial_sum", name).group())
        if re.search(r"rms_bwd_kernelIdd.*Li1024E", name):  # float64 rows of more than 4096 channels
            continue
        assert k[".vgpr_spill_count"] == 0 and k[".private_segment_fixed_size"] == 0, name
    assert seen == {"rms_fwd", "rms_bwd", "rotary", "rotary_norm_bwd", "clip", "partial_sum"}


def test_walks_are_resident(kernels):
    """The backwards walk with two and three workgroups a CU."""
    for name, k in kernels.items():
        if "rms_bwd" in name and "Li256E" in name:
            assert _workgroups_per_cu(k) >= 2, name
        if "rotary_norm_bwd" in name:
            assert _workgroups_per_cu(k) >= 3 or "kernelIdd" in name, name
