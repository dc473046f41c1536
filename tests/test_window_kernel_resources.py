"""CPU checks of what the compiler made of the attention kernels: no register lies in scratch memory (wavefronts count the copies that
they wait for, and an access to scratch memory would be among them), and as many workgroups fit a CU as they are bound for."""
import re

import pytest

from gnnhwc import _cabi
from tests.test_kernel_resources import LDS_PER_CU, TYPES, _kernels, _workgroups_per_cu


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


def _bound(kernel, bytes_of_type, width, last):
    """Workgroups of 256 threads a CU that a kernel is written for; last: FINE of a forward, PARTS of a backward."""
    if kernel == "window_forward":
        return 2 if bytes_of_type == 4 else 4 if width <= 64 and not last else 2 if width <= 128 else 1
    if kernel == "window_dq":
        return 2 if width <= (128 if bytes_of_type == 2 else 96) else 1
    return 2 if (width <= 64 and bytes_of_type == 2) or (bytes_of_type == 4 and last == 1) else 1


def test_as_many_workgroups_fit_a_cu_as_the_kernels_are_bound_for(kernels):
    """The plan counts on them (the workgroups that a CU takes at once), and the figures beside the code were measured with them."""
    seen = set()
    for name, k in kernels.items():
        m = re.search(r"\d+(window_forward|window_dq|window_dkv)_kernelI(DF16_|NS_6bf16_tE|f)Li(\d+)E(?:L[bi](\d)E)?E", name)
        if not m:
            continue
        kernel, type_, width, last = m.group(1), TYPES[m.group(2)], int(m.group(3)), int(m.group(4) or 0)
        seen.add((kernel, type_, width, last))
        assert k[".max_flat_workgroup_size"] == 256
        assert _workgroups_per_cu(k) >= _bound(kernel, 4 if type_ == "f32" else 2, width, last), (name, k[".vgpr_count"], k[".group_segment_fixed_size"])
    assert {s[2] for s in seen} == {64, 96, 128, 160, 256} and len(seen) == (3 + 3 + 4) + 2 * (5 * 2 + 5 + 3 + 2 * 2), sorted(seen)
