"""GPU: row quantisation behind SiLU * up where the sigmoid is below FP32's smallest normal value.

Tolerance: the exponential is good to 2 + 1.173 |x| units in the last place (107 at |x| <= 88.7), the quotient to 2, two more roundings; the
sigmoid itself, from 2.9e-39 on, is held to half of 2^-149: 2^-150 / 2.9e-39 relative."""
import numpy as np
import pytest

import eight_bit_reference as R
from rust_ascend_b200 import B200Runtime as RT
from rust_ascend_b200 import DType, TensorBuffer

pytestmark = pytest.mark.gpu
VALUE = 112 * 2.0 ** -23 + 2.0 ** -150 / 2.9e-39


@pytest.mark.parametrize("width", [64, 301, 4096])
@pytest.mark.parametrize("dtype", [DType.F32, DType.BF16])
@pytest.mark.parametrize("at", [0, 1])
def test_small_sigmoids_of_large_products(client, width, dtype, at):
    """Gates of -85 to -88.7 beside factors of up to 3e38: products of hundreds, which the row's scale follows."""
    rng = np.random.default_rng([width, int(dtype)])
    gate, gv = R.hold(-85 - 3.7 * rng.random((5, width + at)), dtype)
    up, uv = R.hold(rng.standard_normal((5, width + at)) * 7e37, dtype)
    assert gv.min() > -88.72
    view = lambda a: (lambda t: TensorBuffer(t.handle, (5, width), dtype, (width + at, 1), at * dtype.size, t._owner))(client.upload(a, dtype))
    q, s = RT.quantize_rows(client, view(gate), up=view(up))
    R.check_rows(client.read(q), client.read(s), R.silu_mul(gv[:, at:], uv[:, at:]), VALUE + 2 * 2.0 ** -24, VALUE + 4 * 2.0 ** -24)


def test_gates_whose_exponential_overflows_give_zero(client):
    """From -88.8 on, as in rb_silu_mul: exp(-x) is infinite in FP32 and the quotient 0."""
    gate = np.full((2, 48), -89, np.float32)
    gate[0, 3] = 1
    gate[1, 5:] = -1e30
    up = np.full((2, 48), 3e38, np.float32)
    up[0, 3] = 2
    q, s = (client.read(t) for t in RT.quantize_rows(client, client.upload(gate), up=client.upload(up)))
    assert q[0, 3] == 127 and np.abs(q).sum() == 127 and s[1] == np.float32(2.0 ** -126)


@pytest.mark.parametrize("rows,width", [(5, 64), (5, 301), (5, 14336), (5, 30001), (700, 520)])
@pytest.mark.parametrize("dtype", [DType.F32, DType.BF16])
def test_products_near_the_largest_value(client, rows, width, dtype):
    """Rows whose products reach FP32's upper end, beside ordinary ones, one that passes it and one with an infinity."""
    rng = np.random.default_rng([width, int(dtype)])
    gate, up = rng.random((rows, width)) * 6.4, rng.standard_normal((rows, width)) * 3
    up = np.clip(up, -6.4, 6.4)
    up[::5] *= 8e36                # at most 3.3e38
    up[2::5] *= 1e36               # at most 4.1e37: within a quarter of the range
    up[3, 7], gate[3, 7] = 3e38, 2
    gate[4, 1] = np.inf
    gate[0, 3], up[0, 3] = 6.375, 5e37
    (g, gv), (u, uv) = R.hold(gate, dtype), R.hold(up, dtype)
    q, s = (client.read(t) for t in RT.quantize_rows(client, client.upload(g, dtype), up=client.upload(u, dtype)))
    good = np.setdiff1d(np.arange(rows), [3, 4])
    exact = R.silu_mul(gv[good], uv[good])
    assert np.abs(exact[0]).max() > 3e38 and np.isnan(s[3:5]).all() and not q[3:5].any()
    near = 14 * 2.0 ** -23         # gates up to 6.5, as derived in test_quant_gpu
    R.check_rows(q[good], s[good], exact, near + 2 * 2.0 ** -24, near + 4 * 2.0 ** -24)
