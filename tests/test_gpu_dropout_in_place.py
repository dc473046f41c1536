"""GPU tests of gnnhwc_dropout over its own inputs, which the header allows: y may be x, or the residual."""
import ctypes

import pytest
import torch

from gnnhwc import _cabi, dropout
from tests.left_alone import generators_left_alone  # noqa: F401 (a fixture)
from tests.test_gpu_dropout import BF16, F16, F32, F64, normal

pytestmark = pytest.mark.gpu
CODES = {F32: _cabi.F32, F64: _cabi.F64, F16: _cabi.F16, BF16: _cabi.BF16}


@pytest.mark.parametrize("dtype", [F32, F64, F16, BF16])
@pytest.mark.parametrize("n", [1, 2047, 2048, 100003])
def test_over_its_inputs(n, dtype, device):
    x, r = normal((n,), dtype, device, 1), normal((n,), dtype, device, 2)
    for residual, over in ((False, "x"), (True, "x"), (True, "residual")):
        want = dropout(x, 0.3, 7, 5, residual=r if residual else None)
        mine = {"x": x.clone(), "residual": r.clone()}
        stream = ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)
        code = _cabi.lib.gnnhwc_dropout(mine["x"].data_ptr(), mine["residual"].data_ptr() if residual else None, mine[over].data_ptr(), n, 0.3, 7, None, 5, CODES[dtype], stream)
        assert code == 0 and torch.equal(mine[over], want)
        other = "residual" if over == "x" else "x"
        assert torch.equal(mine[other], {"x": x, "residual": r}[other])
