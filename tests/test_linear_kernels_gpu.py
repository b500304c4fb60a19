"""GPU: every kernel of the 8-bit linear, in every form that a call can be sent to, to the bit."""
import pytest

from linear_sizes import SIZES
from rust_ascend_b200 import DType
from test_quant_gpu import linear_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("dtype", [DType.F32, DType.BF16, DType.F16])
def test_linear(client, size, dtype):
    linear_case(client, *size, dtype, bias=dtype != DType.F16, seed=1)
