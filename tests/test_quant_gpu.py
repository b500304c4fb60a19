"""GPU: rows held in 8 bits and the 8-bit linear against their definitions in 64 bits.

Tolerances.  q = rint(v c) with one fused rounding, v = x (exact), s w (one rounding, 2^-24) or SiLU(x) up, c = 127 / max (two
roundings): v c is off by at most 4 x 2^-24 relative, which moves q by that times 127 beyond half a step.  The norm's scale also has the
root: the sum of squares adds at most 64 terms one after the other and then 10 levels of a tree, 74 x 2^-24 relative, halved by the root,
plus 8 roundings around it.  SiLU: the exponential is good to 2 + 1.173 |x| units in the last place (10 at |x| <= 6.5), the quotient to 2,
two more roundings: 14 x 2^-23."""
import numpy as np
import pytest

import eight_bit_reference as R
from rust_ascend_b200 import B200Runtime as RT
from rust_ascend_b200 import DType, TensorBuffer

pytestmark = pytest.mark.gpu
F32, F16, BF16, I8 = DType.F32, DType.F16, DType.BF16, DType.I8
VALUE = 4 * 2.0 ** -24
NORM_SCALE = (37 + 8) * 2.0 ** -24
SILU = 14 * 2.0 ** -23



@pytest.mark.parametrize("rows,width", [(1, 4096), (3, 1), (5, 7), (2, 8), (33, 72), (9, 333), (17, 2049), (301, 4096), (4, 5120), (2, 8193), (2, 16384), (3, 16392), (1, 40001), (700, 128)])
@pytest.mark.parametrize("dtype,wtype", [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)])
@pytest.mark.parametrize("residual", [False, True])
def test_norm_quant(client, rows, width, dtype, wtype, residual):
    rng = np.random.default_rng([rows, width, int(dtype)])
    x, xv = R.hold(rng.standard_normal((rows, width)) * 3, dtype)
    d, dv = R.hold(rng.standard_normal((rows, width)), dtype)
    w, wv = R.hold(1 + 0.2 * rng.standard_normal(width), wtype)
    up = client.upload
    got = RT.rms_norm_quant(client, up(x, dtype), up(w, wtype), 1e-5, delta=up(d, dtype) if residual else None)
    if residual:
        total = R.hold(xv + dv, dtype)[1]             # the FP32 sum, rounded to the storage type
        assert np.array_equal(R.read(client, got[2]), total)
        xv = total
    R.check_rows(client.read(got[0]), client.read(got[1]), R.norm(xv, wv, np.float64(np.float32(1e-5))), NORM_SCALE, VALUE)


def test_norm_quant_agrees_with_the_norms_of_the_framework(client):
    """The rows that rb_add_rms_norm stores, quantised, are the rows of the fused operator (up to the norm's own FP32 roundings)."""
    rng = np.random.default_rng(3)
    x, d = (rng.standard_normal((40, 512)).astype(np.float32) for _ in range(2))
    w = rng.standard_normal(512).astype(np.float32)
    up = client.upload
    q, s, total = RT.rms_norm_quant(client, up(x), up(w), 1e-5, delta=up(d))
    y, _ = RT.rms_norm(client, total, up(w), 1e-5)
    q2, s2 = RT.quantize_rows(client, y)
    assert np.abs(client.read(s) / client.read(s2) - 1).max() <= NORM_SCALE + VALUE
    assert np.abs(client.read(q).astype(int) - client.read(q2)).max() <= 1 and np.mean(client.read(q) != client.read(q2)) < 1e-3


def test_norm_quant_in_place(client):
    rng = np.random.default_rng(4)
    x, d, w = rng.standard_normal((20, 17000)).astype(np.float32), rng.standard_normal((20, 17000)).astype(np.float32), np.ones(17000, np.float32)
    up = client.upload
    want = RT.rms_norm_quant(client, up(x), up(w), 1e-5, delta=up(d))
    stream = up(x)
    q, s = client.tensor((20, 17000), I8), client.tensor((20,), F32)
    RT.rms_norm_quant(client, stream, up(w), 1e-5, delta=up(d), out=(q, s, stream))
    for a, b in zip(want, (q, s, stream)):
        assert np.array_equal(client.read(a), client.read(b))


@pytest.mark.parametrize("rows,width", [(1, 1), (2, 3), (7, 16), (5, 100), (1, 14336), (64, 4096), (129, 1001), (3, 11008), (2, 20003), (1000, 24)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_quantize_rows(client, rows, width, dtype):
    rng = np.random.default_rng([rows, width, int(dtype)])
    x, xv = R.hold(rng.standard_normal((rows, width)) * np.exp(rng.standard_normal((rows, 1)) * 2), dtype)
    q, s = RT.quantize_rows(client, client.upload(x, dtype))
    R.check_rows(client.read(q), client.read(s), xv.astype(np.float64), 2 * 2.0 ** -24, VALUE)


@pytest.mark.parametrize("rows,width", [(1, 8), (3, 5), (6, 128), (8, 14336), (37, 1003), (130, 2560), (2, 30000)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("fused", [False, True])
def test_silu_quantize_rows(client, rows, width, dtype, fused):
    """Gate and up as two tensors, or as the halves of one [rows, 2 width] projection."""
    rng = np.random.default_rng([rows, width, int(dtype)])
    both, bv = R.hold(np.clip(rng.standard_normal((rows, 2 * width)) * 2, -6.5, 6.5), dtype)
    if fused:
        t = client.upload(both, dtype)
        gate = TensorBuffer(t.handle, (rows, width), dtype, (2 * width, 1), 0, t._owner)
        up = TensorBuffer(t.handle, (rows, width), dtype, (2 * width, 1), width * dtype.size, t._owner)
    else:
        gate, up = client.upload(both[:, :width], dtype), client.upload(both[:, width:], dtype)
    q, s = RT.quantize_rows(client, gate, up=up)
    R.check_rows(client.read(q), client.read(s), R.silu_mul(bv[:, :width], bv[:, width:]), SILU + 2 * 2.0 ** -24, SILU + VALUE)


def test_strided_rows_of_rank_three_and_padding_untouched(client):
    rng = np.random.default_rng(8)
    a = rng.standard_normal((3, 5, 40)).astype(np.float32)
    t = client.upload(a)
    view = TensorBuffer(t.handle, (3, 5, 33), F32, (200, 40, 1), 12, t._owner)      # columns 3..35, four-byte aligned rows
    q, s = RT.quantize_rows(client, view)
    assert q.shape == (3, 5, 33) and s.shape == (3, 5)
    R.check_rows(client.read(q), client.read(s), a[:, :, 3:36].astype(np.float64), 2 * 2.0 ** -24, VALUE)
    assert np.array_equal(client.read(t), a)


@pytest.mark.parametrize("width", [16, 33, 4096, 9000])
def test_special_rows(client, width):
    """Zeros, NaN, infinities, values near the ends of FP32, denormal numbers, one large value, exact ties."""
    x = np.zeros((10, width), np.float32)
    x[1, 3] = np.nan
    x[2, 5] = np.inf
    x[3, 1] = -np.inf
    x[4] = np.linspace(-1, 1, width) * 3e38
    x[5] = np.linspace(-1, 1, width) * 1e-36
    x[6] = np.linspace(-1, 1, width) * 1e-40
    x[7, 0], x[7, 1] = 1e30, 1.0
    x[8] = (np.arange(width) % 255 - 127) / 2.0      # 127 / 2 is the largest: every odd number sits between two steps of ... one half
    x[8, 0], x[8, 1] = 127.0, 0.5                    # scale 1: halves are exact ties, to even
    x[9] = 1e-45
    q, s = RT.quantize_rows(client, client.upload(x))
    q, s = client.read(q), client.read(s)
    for r in (1, 2, 3):
        assert np.isnan(s[r]) and not q[r].any()
    assert s[0] == np.float32(2.0 ** -126) and not q[0].any()
    for r in (4, 5, 6, 7, 9):
        want = R.scale_of(x[r:r + 1].astype(np.float64))[0]
        assert abs(s[r] / want - 1) <= 2 * 2.0 ** -24
        assert np.abs(q[r] - x[r].astype(np.float64) / want).max() <= 0.5 + 127 * VALUE
    assert s[8] == 1.0 and np.array_equal(q[8], np.rint(x[8]).astype(np.int8))
    y = client.read(RT.dequantize_rows(client, client.upload(q), client.upload(s), F32))
    assert np.isnan(y[1:4]).all() and not y[0].any()


def test_special_rows_of_the_norm(client):
    width = 256
    x = np.zeros((6, width), np.float32)
    x[1, 3] = np.nan
    x[2, 5] = -np.inf
    x[3] = 1e-30
    x[4] = 1e25                                       # the sum of squares overflows: the norm is zero, as in rb_rms_norm
    x[5, 0] = 7.0
    w = np.full(width, 1.5, np.float32)
    q, s = RT.rms_norm_quant(client, client.upload(x), client.upload(w), 1e-6)
    q, s = client.read(q), client.read(s)
    assert np.isnan(s[1]) and np.isnan(s[2]) and not q[1].any() and not q[2].any()
    assert not q[0].any() and s[0] == np.float32(2.0 ** -126)
    assert (q[3] == 127).all() and not q[4].any() and q[5, 0] == 127 and not q[5, 1:].any()
    w0 = np.zeros(width, np.float32)
    q, s = RT.rms_norm_quant(client, client.upload(x[5:]), client.upload(w0), 1e-6)
    assert not client.read(q).any() and client.read(s)[0] == np.float32(2.0 ** -126)


@pytest.mark.parametrize("rows,width", [(1, 1), (3, 5), (2, 16), (31, 33), (100, 4096), (7, 1000), (5, 20003)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_dequantize_rows(client, rows, width, dtype):
    rng = np.random.default_rng([rows, width])
    q = rng.integers(-128, 128, (rows, width)).astype(np.int8)
    s = rng.uniform(0.001, 0.1, rows).astype(np.float32)
    y = RT.dequantize_rows(client, client.upload(q), client.upload(s), dtype)
    assert np.array_equal(R.read(client, y), R.hold(q.astype(np.float32) * s[:, None], dtype)[1])


# ---- the linear: integer sums are exact, so every rounding is known and results have to match to the bit -----------------------
def linear_case(client, m, n, k, dtype, bias, seed=0, extreme=False):
    rng = np.random.default_rng([m, n, k, seed])
    x = rng.integers(-128, 128, (m, k)).astype(np.int8)
    w = rng.integers(-128, 128, (n, k)).astype(np.int8)
    if extreme:
        x[:], w[:] = -128, -128
        w[1::2] = 127
    sx, sw = rng.uniform(0.001, 0.1, m).astype(np.float32), rng.uniform(0.0001, 0.01, n).astype(np.float32)
    b = rng.standard_normal(n).astype(np.float32) if bias else None
    up = client.upload
    y = RT.linear_i8(client, up(x), up(sx), up(w), up(sw), bias=None if b is None else up(b), dtype=dtype)
    acc = x.astype(np.float64) @ w.astype(np.float64).T          # below 2^53: exact
    want = acc.astype(np.float32) * (sx[:, None] * sw[None, :])
    if bias:
        want = want + b
    assert np.array_equal(R.read(client, y), R.hold(want, dtype)[1])


@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 33, 64, 65, 100, 128, 129, 257, 500, 513, 777])
@pytest.mark.parametrize("n,k", [(128, 128), (1, 16), (129, 144), (257, 1040), (1000, 4096)])
def test_linear_sizes(client, m, n, k):
    linear_case(client, m, n, k, BF16, bias=False)


@pytest.mark.parametrize("m,n,k", [(1, 4096, 4096), (8, 300, 16384), (40, 1001, 2064), (300, 515, 528), (1025, 2051, 784), (2048, 1536, 512)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("bias", [False, True])
def test_linear_types(client, m, n, k, dtype, bias):
    linear_case(client, m, n, k, dtype, bias)


@pytest.mark.parametrize("m,n,k", [(3, 65, 16), (4, 65, 4112), (5, 65, 16), (5, 4705, 1168), (5, 67, 880), (5, 67, 944), (18, 9473, 16), (17, 5183, 1744), (17, 2201, 960),
                                   (18, 995, 912), (33, 9603, 16), (35, 5155, 3232), (35, 2867, 1824), (33, 1671, 1456), (390, 11055, 16), (65, 9523, 16), (68, 6307, 4928),
                                   (68, 3129, 2880), (70, 1867, 2800), (194, 9797, 16), (600, 5003, 2064)])
def test_linear_of_every_tile_and_split(client, m, n, k):
    """Sizes at which each tile width with each split of K is the quickest, with ragged edges in all three directions."""
    linear_case(client, m, n, k, BF16, bias=True)


@pytest.mark.parametrize("m", [1, 20, 600])
def test_linear_largest_sums(client, m):
    """-128 times -128 over the largest K is the largest sum that 32 bits hold."""
    linear_case(client, m, 130, 131056, F32, bias=False, extreme=True)


def test_linear_many_column_tiles_and_tail(client):
    linear_case(client, 700, 19456 + 77, 256, BF16, bias=True)


def test_linear_of_nan_rows_and_leading_axes(client):
    """A row whose scale is NaN (quantised from a NaN) gives NaN; the others are untouched.  Rank 3 keeps its leading axes."""
    rng = np.random.default_rng(1)
    x = rng.integers(-127, 128, (2, 3, 64)).astype(np.int8)
    w = rng.integers(-127, 128, (40, 64)).astype(np.int8)
    sx = np.full((2, 3), 0.5, np.float32)
    sx[1, 1] = np.nan
    y = RT.linear_i8(client, client.upload(x), client.upload(sx), client.upload(w), client.upload(np.ones(40, np.float32)), dtype=F32)
    assert y.shape == (2, 3, 40)
    y = client.read(y)
    want = (x.astype(np.int64) @ w.astype(np.int64).T).astype(np.float32) * sx[..., None]
    assert np.isnan(y[1, 1]).all() and np.array_equal(y, want, equal_nan=True)


def test_linear_respects_the_sm_limit(client):
    import ctypes as C
    from rust_ascend_b200.runtime import _check
    _check(client._lib.rb_set_sm_limit(client._ctx, C.c_int32(20)))
    try:
        linear_case(client, 900, 1200, 256, BF16, bias=False)
        linear_case(client, 4, 1200, 256, BF16, bias=False)
    finally:
        _check(client._lib.rb_set_sm_limit(client._ctx, C.c_int32(0)))


def test_more_than_2_to_the_32_values(client):
    """Offsets beyond 32 bits in every operator: 4.6e9 values, of which the last row is checked."""
    rows, width = 70000, 65536
    rng = np.random.default_rng(1)
    x = client.tensor((rows, width), F16)
    client.memset(x, 0)
    last = rng.standard_normal(width).astype(np.float16)
    client.write(x.handle, last, (rows - 1) * width * 2)
    client.sync()
    q, s = RT.quantize_rows(client, x)
    lq = np.empty(width, np.int8)
    client.read_into(q.handle, lq, (rows - 1) * width)
    ls = client.read(s)[-1:]
    R.check_rows(lq[None], ls, last.astype(np.float64)[None], 2 * 2.0 ** -24, VALUE)
    w = client.upload(np.ones(width, np.float32))
    q2, s2 = RT.rms_norm_quant(client, x, w, 1e-5, out=(q,))
    client.read_into(q.handle, lq, (rows - 1) * width)
    R.check_rows(lq[None], client.read(s2)[-1:], R.norm(last[None], np.ones(width), 1e-5), NORM_SCALE, VALUE)
    RT.dequantize_rows(client, q, s2, out=x)
    back = np.empty(width, np.float16)
    client.read_into(x.handle, back, (rows - 1) * width * 2)
    assert np.array_equal(back, (lq.astype(np.float32) * client.read(s2)[-1]).astype(np.float16))
    del q, q2, s, s2
    # y of 70000 x 65536 from K = 32: the last rows and columns
    a, b = rng.integers(-127, 128, (rows, 32)).astype(np.int8), rng.integers(-127, 128, (width, 32)).astype(np.int8)
    one = lambda n: client.upload(np.ones(n, np.float32))
    RT.linear_i8(client, client.upload(a), one(rows), client.upload(b), one(width), out=x)
    client.read_into(x.handle, back, (rows - 1) * width * 2)
    with np.errstate(over="ignore"):
        assert np.array_equal(back, (b.astype(np.float32) @ a[-1].astype(np.float32)).astype(np.float16))


@pytest.mark.parametrize("width", [256, 301, 1000, 5003, 8192, 8193, 12000, 16384, 16390])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_silu_rows_that_start_anywhere(client, width, dtype):
    """Gate and up at any element of wider rows, each at another distance from a 16-byte boundary: what aligned rows give, bit for bit."""
    rng = np.random.default_rng([width, int(dtype)])
    rows = 7
    gate, gv = R.hold(np.clip(rng.standard_normal((rows, width)) * 2, -6.5, 6.5), dtype)
    up, uv = R.hold(np.clip(rng.standard_normal((rows, width)) * 2, -6.5, 6.5), dtype)
    per = 16 // dtype.size
    wanted = R.silu_mul(gv, uv)
    first = None
    for at, far in ((0, 0), (1, 0), (0, per - 1), (3, 2), (per - 1, 1)):
        pitch = (2 * width + 64) // per * per + (per + 1 if at % 2 else 0)
        wide = np.zeros((rows, pitch), gate.dtype)
        second = (width + 2 * per) // per * per + far
        wide[:, at:at + width], wide[:, second:second + width] = gate, up
        t = client.upload(wide, dtype)
        view = lambda start: TensorBuffer(t.handle, (rows, width), dtype, (pitch, 1), start * dtype.size, t._owner)
        q, s = RT.quantize_rows(client, view(at), up=view(second))
        got = client.read(q), client.read(s)
        R.check_rows(*got, wanted, SILU + 2 * 2.0 ** -24, SILU + VALUE)
        first = first or got
        assert np.array_equal(got[0], first[0]) and np.array_equal(got[1], first[1])
        assert np.array_equal(client.read(t), wide)


@pytest.mark.parametrize("width", [303, 5001, 9001])
def test_special_values_in_silu_rows_that_start_anywhere(client, width):
    rng = np.random.default_rng(width)
    g, u = rng.standard_normal((7, width)).astype(np.float32), rng.standard_normal((7, width)).astype(np.float32)
    g[1, 2], u[2, width - 1], g[3, width // 2] = np.nan, np.inf, np.inf
    g[4], u[5] = 0, 0
    u[6] *= 1e-30                                         # values that are raised before they are divided
    q, s = (client.read(t) for t in RT.quantize_rows(client, client.upload(g), up=client.upload(u)))
    assert np.isnan(s[1:4]).all() and not q[1:6].any() and np.all(s[4:6] == np.float32(2.0 ** -126))
    R.check_rows(q[[0, 6]], s[[0, 6]], R.silu_mul(g[[0, 6]], u[[0, 6]]), SILU + 2 * 2.0 ** -24, SILU + VALUE)


@pytest.mark.parametrize("rows,width", [(3, 4), (9, 1032), (170, 5000), (300, 2056), (5, 20008), (160, 1004)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("residual", [False, True])
def test_norm_rows_that_end_inside_a_round(client, rows, width, dtype, residual):
    """Widths whose last vectors fill only some lanes of a warp, with the sum written over the input."""
    rng = np.random.default_rng([rows, width, int(dtype), residual])
    x, xv = R.hold(rng.standard_normal((rows, width)), dtype)
    d, dv = R.hold(rng.standard_normal((rows, width)), dtype)
    w, wv = R.hold(1 + 0.2 * rng.standard_normal(width), dtype)
    t, wt = client.upload(x, dtype), client.upload(w, dtype)
    total = xv
    if residual:
        total = R.hold(xv + dv, dtype)[1]
        q, s, stored = RT.rms_norm_quant(client, t, wt, 1e-5, delta=client.upload(d, dtype), out=(None, None, t))
        assert np.array_equal(R.read(client, stored), total)
    else:
        q, s = RT.rms_norm_quant(client, t, wt, 1e-5)
    R.check_rows(client.read(q), client.read(s), R.norm(total, wv, 1e-5), NORM_SCALE, VALUE)
