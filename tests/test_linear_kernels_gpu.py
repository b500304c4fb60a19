"""GPU: every kernel of the 8-bit linear, in every form that a call can be sent to, to the bit; which one runs, and on how many SMs."""
import ctypes as C

import pytest

from launched import launched
from linear_sizes import SIZES
from rust_ascend_b200 import B200Runtime as RT
from rust_ascend_b200 import DType
from rust_ascend_b200.runtime import _check
from test_quant_gpu import linear_case

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def limit(client):
    """Sets the context's SM limit.  Every test here begins and ends without one, whatever was set before."""
    def set_to(sms):
        _check(client._lib.rb_set_sm_limit(client._ctx, C.c_int32(sms)))
    set_to(0)
    yield set_to
    set_to(0)


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("dtype", [DType.F32, DType.BF16, DType.F16])
def test_linear(client, size, dtype):
    linear_case(client, *size, dtype, bias=dtype != DType.F16, seed=1)


def kernel_of(client, m, n, k):
    t = client.tensor
    x, sx, w, sw, y = t((m, k), DType.I8), t((m,), DType.F32), t((n, k), DType.I8), t((n,), DType.F32), t((m, n), DType.BF16)
    for a in (x, sx, w, sw):
        client.memset(a, 0)

    def call():
        RT.linear_i8(client, x, sx, w, sw, out=y)
    call()
    (name, blocks), = launched(client, call)
    assert "linear_i8" in name
    return next(kind for kind in ("row", "few", "pair") if f"linear_i8_{kind}_kernel" in name), blocks


@pytest.mark.parametrize("size", SIZES, ids=str)
def test_the_kernel_that_runs(client, size):
    assert kernel_of(client, *size)[0] == SIZES[size][0].rstrip("s")


# one call for each kernel and some that fill the GPU, ragged ones among them
LIMITED = [(1, 6145, 4096), (1, 70, 4096), (3, 65, 16), (2, 3000, 528), (5, 67, 944), (17, 2201, 960), (33, 1671, 1456), (130, 4100, 784), (900, 1200, 256), (512, 4096, 4096), (2048, 4096, 512)]


@pytest.mark.parametrize("sms", [2, 3, 20, 100, 147])
def test_sm_limit(client, limit, sms):
    """No call has more CTAs than the limit, so it cannot occupy more SMs; results are what they are without one."""
    for m, n, k in LIMITED:
        limit(sms)
        kind, blocks = kernel_of(client, m, n, k)
        assert blocks <= sms, (m, n, k, kind, blocks)
        linear_case(client, m, n, k, DType.BF16, bias=True, seed=sms)


def test_smallest_limit_and_one_that_limits_nothing(client, limit):
    limit(1)
    assert kernel_of(client, 900, 1200, 256) == ("pair", 2)          # a pair is the least that the kernel for many tokens runs on
    assert kernel_of(client, 5, 67, 944) == ("few", 1)
    linear_case(client, 900, 1200, 256, DType.BF16, bias=True)
    limit(client.properties()["sm_count"])
    assert kernel_of(client, 18, 9473, 16)[0] == "few"
