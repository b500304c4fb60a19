"""GPU: log probabilities of given tokens, entropy, top alternatives and their gradient against the definitions in 64 bits.

Tolerance of ln S.  A term 2^d is off by 2^-22 (the exponential) and by ln2 |d| 3 x 2^-24 (d's roundings); weighted with its share of the
sum, the |d| are at most about log2 of the vocabulary (17).  A thread adds at most V / 256 + 16 terms one after the other (one rounding
each), then 8 + 3 levels.  So |ln S| is off by D = 2^-22 + 17 ln2 3 x 2^-24 + (V / 256 + 27) x 2^-24 at most, T / S by that times 18 more.
A log probability adds the roundings of scale (x - M) (three, relative); lse that of its result."""
import numpy as np
import pytest

import eight_bit_reference as R
from rust_ascend_b200 import B200Runtime as RT
from rust_ascend_b200 import DType, TensorBuffer

pytestmark = pytest.mark.gpu
F32, F16, BF16, I32 = DType.F32, DType.F16, DType.BF16, DType.I32
U = 2.0 ** -24


def spread(vocab):
    return 2.0 ** -22 + 17 * 0.7 * 3 * U + (vocab / 256 + 27) * U


def compare(got, want, vocab, top):
    log_prob, lse, entropy, values, ids = got
    w_log_prob, w_lse, w_entropy, w_values, w_ids, _ = want
    d = spread(vocab)
    with np.errstate(invalid="ignore", over="ignore"):
        for a, w, extra in ((log_prob, w_log_prob, 0), (lse, w_lse, 0), (entropy, w_entropy, 20 * d)) + (((values, w_values, 0),) if top else ()):
            same = (np.isnan(a) & np.isnan(w)) | (a == w) | (np.isinf(a) & (a == w.astype(np.float32)))      # beyond FP32's range the rounded result is infinite
            off = np.where(same, 0, np.abs(a - w) - (d + extra + 6 * U * np.abs(w)))
            assert off.max(initial=0) <= 0, off.max()
    if top:
        assert np.array_equal(ids, w_ids)


def call(client, x, xv, ids, dtype, scale, top, ignore=-100, view=None):
    t = view if view is not None else client.upload(x, dtype)
    out = RT.token_log_probs(client, t, client.upload(ids), scale=scale, ignore_index=ignore, top_k=top)
    compare([None if o is None else client.read(o) for o in out], R.scores(xv, ids, scale, ignore, top), xv.shape[1], top)
    return t, out


def case(rows, vocab, dtype, seed=0, spread_of=2.5):
    rng = np.random.default_rng([rows, vocab, seed])
    x, xv = R.hold(rng.standard_normal((rows, vocab)) * spread_of, dtype)
    ids = rng.integers(0, vocab, rows)
    ids[rng.random(rows) < 0.2] = -100
    return rng, x, xv, ids


@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 2, 2), (2, 7, 3), (5, 64, 64), (4, 257, 20), (7, 1000, 1), (3, 8192, 64), (1, 32000, 20), (2, 50001, 64), (1, 128000, 33),
                                            (9, 4099, 5), (300, 3001, 7), (700, 515, 0), (40, 20011, 10)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_scores(client, rows, vocab, top, dtype):
    rng, x, xv, ids = case(rows, vocab, dtype)
    call(client, x, xv, ids, dtype, 1.25, top)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("pad,offset", [(1, 0), (64, 0), (5, 3)])
def test_padded_rows_and_unaligned_starts(client, dtype, pad, offset):
    rng, x, xv, ids = case(6, 5000 + pad, dtype)
    x[:, :offset] = x[:, 5000 + offset:] = np.array(60000.0 if dtype != BF16 else 0x477f).astype(x.dtype)      # a large value: reading it would show
    t = client.upload(x, dtype)
    view = TensorBuffer(t.handle, (6, 5000 - offset), dtype, (5000 + pad, 1), offset * dtype.size, t._owner)
    call(client, None, xv[:, offset:5000], np.where(ids >= 5000 - offset, 0, ids), dtype, 1.0, 8, view=view)


@pytest.mark.parametrize("vocab", [100, 5000, 40000])
@pytest.mark.parametrize("top", [0, 20, 64])
def test_masked_and_special_rows(client, vocab, top):
    """Masks by -inf and by the type's lowest value, rows without any logit, NaN, +inf, constant rows, both zeros, a single survivor."""
    rng = np.random.default_rng(vocab + top)
    x = (rng.standard_normal((12, vocab)) * 2).astype(np.float32)
    keep = rng.integers(0, vocab, 5)
    for r, masked in ((0, -np.inf), (1, np.finfo(np.float32).min)):
        row = np.full(vocab, masked, np.float32)
        row[keep] = x[r, keep]
        x[r] = row
    x[2] = -np.inf
    x[3, vocab // 3] = np.nan
    x[4, vocab // 2] = np.inf
    x[5] = 1.5
    x[6] = 0.0
    x[6, ::3] = -0.0
    x[7] = -np.inf
    x[7, vocab - 1] = -4.0
    x[8] = np.arange(vocab)[::-1] * 1e-3
    x[9] = np.arange(vocab) * 1e-3
    x[10] = np.round(x[10])                           # many ties everywhere
    x[11] = np.finfo(np.float32).min
    ids = rng.integers(0, vocab, 12)
    ids[0], ids[7] = keep[0], vocab - 1
    ids[11] = -100
    call(client, x, x, ids, F32, 0.7, top)


def test_hostile_order_for_the_top_list(client):
    """The largest values sit in few slices of every split, far more of them than are asked for."""
    vocab = 60000
    x = np.random.default_rng(0).standard_normal((4, vocab)).astype(np.float32)
    for r, period in enumerate((256 * 4, 2048, 8, 512)):
        at = np.arange(vocab) % period < 8
        x[r, at] += 100
    ids = np.zeros(4, np.int64)
    call(client, x, x, ids, F32, 1.0, 64)
    x, xv = R.hold(x, BF16)
    call(client, x, xv, ids, BF16, 1.0, 17)


@pytest.mark.parametrize("rows,vocab", [(3, 30000), (640, 5000)])
@pytest.mark.parametrize("offset,width", [(1000.0, 0.5), (-300.0, 0.01), (64.0, 1e-4), (1.9, 0.3), (0.0, 1e-30)])
def test_logits_close_together(client, rows, vocab, offset, width):
    """Rows whose largest values share many leading bits, and rows around a power of two."""
    rng = np.random.default_rng([rows, int(width * 1e4)])
    x = (offset + rng.standard_normal((rows, vocab)) * width).astype(np.float32)
    call(client, x, x, rng.integers(0, vocab, rows), F32, 1.0, 20)


def test_ids_outside_the_vocabulary_and_other_ignore_index(client):
    rng, x, xv, ids = case(8, 300, F32)
    ids[:4] = (300, -1, 2**40, 7)
    call(client, x, xv, ids, F32, 1.0, 2, ignore=7)
    call(client, x, xv, np.where(np.abs(ids) > 2**31 - 1, 300, ids).astype(np.int32), F32, 1.0, 2, ignore=7)


def test_outputs_may_be_left_out_and_neighbours_stay(client):
    rng, x, xv, ids = case(5, 777, F32)
    t, i = client.upload(x), client.upload(ids)
    full = RT.token_log_probs(client, t, i)
    out = [client.tensor((5,), F32), client.tensor((5,), F32), None]
    RT.token_log_probs(client, t, i, out=out)
    for a, b in zip(full[:2], out):
        assert np.array_equal(client.read(a), client.read(b))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("vocab,top,pad", [(70, 0, 0), (70, 7, 3), (70, 64, 0), (3001, 1, 0), (3001, 32, 1), (3001, 33, 0), (3001, 64, 5), (9000, 5, 8), (34000, 0, 0), (34000, 20, 1)])
def test_many_rows(client, dtype, vocab, top, pad):
    """More rows than blocks of the larger kind fit the GPU, ordinary ones among masked, constant, tied, ascending and special ones."""
    rows = 700 if vocab < 30000 else 610
    rng, x, _, ids = case(rows, vocab + pad, dtype, seed=3)
    rows_of = lambda n: slice(n, None, 40)
    low = {F32: np.float32(np.finfo(np.float32).min), BF16: np.uint16(0xff7f), F16: np.float16(-65504)}[dtype]
    inf, nan = {F32: (np.float32(np.inf), np.float32(np.nan)), BF16: (np.uint16(0x7f80), np.uint16(0x7fc0)), F16: (np.float16(np.inf), np.float16(np.nan))}[dtype]
    minus = np.uint16(0xff80) if dtype == BF16 else -inf
    x[rows_of(1), vocab // 2:] = minus
    x[rows_of(2), vocab // 3:] = low
    x[rows_of(3)] = x[3, 0]
    x[rows_of(4)] = minus
    x[rows_of(5), 5] = nan
    x[rows_of(6), 9] = inf
    x[rows_of(7)] = np.sort(x[rows_of(7)] if dtype != BF16 else x[rows_of(7)] & 0x7fff)
    x[rows_of(8), ::2] = x[8, 0]
    values = {F32: lambda a: a, F16: lambda a: a.astype(np.float32), BF16: R.bf16_bits_to_f32}[dtype](x)[:, :vocab]
    t = client.upload(x, dtype)
    view = TensorBuffer(t.handle, (rows, vocab), dtype, (vocab + pad, 1), 0, t._owner)
    call(client, None, values, np.where(ids >= vocab, 0, ids), dtype, 1.25, top, view=view)


# ---- gradient --------------------------------------------------------------------------------------------------------------------
def gradient_error(xv, ids, scale, g, h, dtype):
    """How far an element may be off: p by the exponential, z - lse and the saved lse, the bracket by its roundings, the result by its storage."""
    _, lse, entropy, _, _, live = R.scores(xv, ids, scale, -100, 0)
    z = xv.astype(np.float64) * scale
    lp = z - lse[:, None]
    p = np.exp(lp)
    d = spread(xv.shape[1])
    bracket = np.abs(np.where(live, g, 0))[:, None] + np.abs(h)[:, None] * (np.abs(np.where(p > 0, lp, 0)) + np.abs(entropy)[:, None])
    rel = 2.0 ** -21 + 4 * U * (np.abs(np.where(p > 0, z, 0)) + np.abs(lse)[:, None]) + d
    return scale * (p * bracket * (rel + 8 * U) + p * np.abs(h)[:, None] * (22 * d) + 4 * U * np.abs(np.where(live, g, 0))[:, None] * p) + 2.0 ** -140


@pytest.mark.parametrize("rows,vocab", [(1, 1), (2, 5), (7, 1000), (33, 4097), (5, 20011), (2, 128000), (600, 300)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("with_entropy", [False, True])
def test_gradient(client, rows, vocab, dtype, with_entropy):
    rng, x, xv, ids = case(rows, vocab, dtype)
    g, h = rng.standard_normal(rows).astype(np.float32), (rng.standard_normal(rows) * 0.3).astype(np.float32) * with_entropy
    t, out = call(client, x, xv, ids, dtype, 1.25, 0)
    up = client.upload
    d = RT.token_log_probs_backward(client, t, up(ids), out[1], out[2] if with_entropy else None, up(g), up(h) if with_entropy else None, scale=1.25)
    got, want = R.read(client, d), R.scores_gradient(xv, ids, 1.25, -100, g, h)
    half = R.half_step(dtype)
    smallest = {F32: 2.0 ** -149, BF16: 2.0 ** -133, F16: 2.0 ** -24}[dtype]
    off = np.abs(got - want) - (gradient_error(xv, ids, 1.25, g, h, dtype) * (1 + half) + (half + 6 * U) * np.abs(want) + smallest)
    assert off.max() <= 0, off.max()
    # in place, and with rows of another alignment
    copy = up(x, dtype)
    RT.token_log_probs_backward(client, copy, up(ids), out[1], out[2], up(g), up(h), scale=1.25, out=copy)
    again = RT.token_log_probs_backward(client, t, up(ids), out[1], out[2], up(g), up(h), scale=1.25)
    assert np.array_equal(R.read(client, copy), R.read(client, again))
    wide = up(np.zeros((rows, vocab + 3), x.dtype), dtype)
    view = TensorBuffer(wide.handle, (rows, vocab), dtype, (vocab + 3, 1), dtype.size, wide._owner)
    RT.token_log_probs_backward(client, t, up(ids), out[1], out[2], up(g), up(h), scale=1.25, out=view)
    held = R.read(client, wide)
    assert np.array_equal(held[:, 1:vocab + 1], R.read(client, again)) and not held[:, 0].any() and not held[:, vocab + 1:].any()


def test_gradient_against_differences(client):
    """Central differences of the 64-bit scores along random directions.  A difference over 2e-4 leaves an error of its square (the third
    derivative is of order one) times the direction's norm; the gradient's own FP32 error is below 1e-5 of the same norm."""
    rng, x, xv, ids = case(4, 500, F32, seed=5)
    g, h = rng.standard_normal(4).astype(np.float32), rng.standard_normal(4).astype(np.float32)
    t, out = call(client, x, xv, ids, F32, 0.8, 0)
    d = client.read(RT.token_log_probs_backward(client, t, client.upload(ids), out[1], out[2], client.upload(g), client.upload(h), scale=0.8)).astype(np.float64)

    def loss(v):
        chosen, _, entropy, _, _, _ = R.scores(v, ids, 0.8, -100, 0)
        return (g * chosen + h * entropy).sum()
    for _ in range(6):
        u = rng.standard_normal(x.shape)
        step = 2e-4
        want = (loss(x + step * u) - loss(x - step * u)) / (2 * step)
        assert abs((d * u).sum() - want) <= 1e-5 * np.linalg.norm(u) + 1e-6


def test_gradient_of_masked_and_idle_rows(client):
    vocab = 3000
    rng = np.random.default_rng(2)
    x = rng.standard_normal((6, vocab)).astype(np.float32)
    x[0, 10:] = -np.inf
    x[1, ::2] = np.finfo(np.float32).min
    x[2] = np.nan                                     # ignored and without upstream: padding may hold anything
    x[3] = -np.inf                                    # scored: NaN
    x[5] = np.nan
    x = np.concatenate([x, np.full((1, vocab), np.finfo(np.float32).min, np.float32)])     # nothing but the mask's value: lse cannot hold it
    ids = np.array([3, 1, -100, 5, -100, 4, 2])
    g = np.array([1, -2, 3, 1, 1, 0, 1], np.float32)
    h = np.array([0.5, 0.25, 0, 0, 0, 0, 0], np.float32)
    out = RT.token_log_probs(client, client.upload(x), client.upload(ids))
    d = client.read(RT.token_log_probs_backward(client, client.upload(x), client.upload(ids), out[1], out[2], client.upload(g), client.upload(h)))
    want = R.scores_gradient(x[:2], ids[:2], 1.0, -100, g[:2], h[:2])
    assert np.abs(d[:2] - want).max() <= 1e-5 and not d[0, 10:].any() and not d[1, ::2].any()
    assert not d[2].any() and np.isnan(d[3]).all() and not d[4].any() and not d[5].any() and np.isnan(d[6]).all()


def test_synchronous_context_reports_a_bad_id():
    """The error of an id outside the vocabulary, in a process of its own: a context is synchronous for its whole life."""
    import subprocess
    import sys
    code = ("import numpy as np\n"
            "from rust_ascend_b200 import B200Runtime as RT, InvalidTensor, RuntimeOptions\n"
            "c = RT.client(RT.initialize_exclusive(RuntimeOptions(0, True)))\n"
            "x = c.upload(np.zeros((2, 50), np.float32))\n"
            "RT.token_log_probs(c, x, c.upload(np.array([3, -100])))\n"
            "try:\n    RT.token_log_probs(c, x, c.upload(np.array([50, 1])))\n"
            "except InvalidTensor as e:\n    print('refused:', e)\n")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "refused: token log probabilities: an id is outside" in r.stdout, r.stdout + r.stderr


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("scale", [1e-30, 1e-18, 1e-3, 0.02, 50.0, 1e9, 1e18, 1e30])
def test_scales_far_from_one(client, dtype, scale):
    """Nearly uniform and nearly certain distributions; all of it in range of FP32 (1e30 times 10 is)."""
    rng, x, xv, ids = case(4, 3001, dtype)
    x[1, 2000:] = np.array(-np.inf, np.float32).astype(np.float16).view(x.dtype) if dtype == F16 else (0xff80 if dtype == BF16 else -np.inf)
    xv = xv.copy()
    xv[1, 2000:] = -np.inf
    ids[1] = 5
    call(client, x, xv, ids, dtype, float(np.float32(scale)), 6)


def test_more_than_2_to_the_32_logits(client):
    """Offsets beyond 32 bits: rows at the end of a batch of 5.2e9 logits, read and written in place."""
    import ctypes as C
    from rust_ascend_b200.runtime import _check
    rows, vocab = 40960, 128000
    t = client.tensor((rows, vocab), BF16)
    client.memset(t, 0)
    ids = np.full(rows, 7, np.int32)
    rng = np.random.default_rng(0)
    bits, last = R.hold(rng.standard_normal(vocab) * 2, BF16)
    client.write(t.handle, bits, (rows - 1) * vocab * 2)
    client.sync()
    i = client.upload(ids)
    out = RT.token_log_probs(client, t, i, top_k=3)
    want = R.scores(last[None], ids[-1:], 1.0, -100, 3)
    got = [client.read(o) for o in out]
    compare([g[-1:] for g in got], want, vocab, 3)
    even = np.log(vocab)
    assert np.abs(got[0][:-1] + even).max() < 1e-4 and np.abs(got[2][:-1] - even).max() < 1e-4 and (got[4][:-1] == [0, 1, 2]).all()
    g = client.upload(np.ones(rows, np.float32))
    RT.token_log_probs_backward(client, t, i, out[1], out[2], g, out=t)
    row = np.empty(vocab, np.uint16)
    client.read_into(t.handle, row, (rows - 1) * vocab * 2)
    d = R.scores_gradient(last[None], ids[-1:], 1.0, -100, np.ones(1), np.zeros(1))[0]
    assert np.abs(R.bf16_bits_to_f32(row) - d).max() <= 2.0 ** -8
    client.read_into(t.handle, row, (rows - 2) * vocab * 2)
    d = R.bf16_bits_to_f32(row)
    assert abs(d[7] - (1 - 1 / vocab)) <= 2.0 ** -8 and np.abs(np.delete(d, 7) * vocab + 1).max() <= 2.0 ** -7


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("vocab", [3000, 130000])
def test_more_ties_than_candidates(client, dtype, vocab):
    """Thousands of equal logits, positive, negative and masked, around the place where the list ends: the lowest indices win."""
    rng = np.random.default_rng(vocab)
    x = np.full((6, vocab), -1.5, np.float32)
    x[1] = 2.25
    x[2] = -np.inf
    x[2, rng.integers(0, vocab, 30)] = rng.standard_normal(30)
    x[3] = rng.integers(-3, 4, vocab)
    x[4] = -rng.integers(5, 9, vocab)
    x[5] = np.where(np.arange(vocab) % 2048 < 1500, -3.0, -4.0)
    x, xv = R.hold(x, dtype)
    for top in (1, 20, 64):
        call(client, x, xv, rng.integers(0, vocab, 6), dtype, 1.0, top)


@pytest.mark.parametrize("dtype,scale,top", [(BF16, 1.0, 1003520.0), (BF16, 1.0, -1003520.0), (BF16, 1.0, 266240.0), (BF16, 0.25, -2129920.0), (F16, 64.0, 65504.0),
                                             (F32, 1.0, 1003520.0), (F32, 64.0, -65504.0)])
def test_gradient_of_certain_rows_far_from_zero(client, dtype, scale, top):
    """One logit far above all others, and lse so large that neighbouring values of the type are hundreds apart: p is 1 there and 0 everywhere
    else, to the bit.  Where it is 1 it inherits the rounding of lse log2(e) (2^-24) and of lse (2^-24, exact here), and the exponential's 2^-22."""
    vocab = 1001
    x = np.full((2, vocab), top - abs(top) / 64)
    x[:, 77] = top
    x[:, 5] = -top if top > 0 else 1.5 * top
    x, xv = R.hold(x, dtype)
    assert xv[0, 77] == top and np.sort(xv[0])[-2] < top
    lse = np.full(2, top * scale, np.float32)
    ids, g, h = np.array([77, 300]), np.array([2, 2], np.float32), np.array([0, 1], np.float32)
    up = client.upload
    d = R.read(client, RT.token_log_probs_backward(client, up(x, dtype), up(ids), up(lse), up(np.zeros(2, np.float32)), up(g), up(h), scale=scale)).astype(np.float64) / scale
    others = np.ones(vocab, bool)
    others[[77, 300]] = False
    assert not d[:, others].any() and d[0, 300] == 0 and d[1, 300] == 2
    # d of the largest: within e of 0, p within exp(e ln 2), and h p log p within h e
    e = 2 * abs(top * scale) * U + 2.0 ** -20
    assert abs(d[0, 77]) <= 2 * np.expm1(e) and abs(d[1, 77] + 2) <= (2 + e) * np.exp(e) * (1 + R.half_step(dtype)) - 2 + 4 * U


def test_rows_written_meanwhile_leave_everything_else_alone(client):
    """Logits that another stream overwrites during the call, ties by random values and back: the scores of that call mean nothing, but it
    stays within its tables and tensors, and the next call is right."""
    import ctypes as C
    from rust_ascend_b200.runtime import _check
    rng = np.random.default_rng(8)
    rows, vocab, top = 150, 40000, 20
    xv = rng.standard_normal((rows, vocab)).astype(np.float32)
    ids = rng.integers(0, vocab, rows)
    ties, values, x, i = client.upload(np.zeros_like(xv)), client.upload(xv), client.upload(np.zeros_like(xv)), client.upload(ids)
    out = [client.tensor((rows,), F32) for _ in range(3)] + [client.tensor((rows, top), F32), client.tensor((rows, top), I32)]
    lib, ctx = client._lib, client._ctx

    def copy(a):
        _check(lib.rb_copy(ctx, C.byref(a._c()), C.byref(x._c())))
    for n in range(40):
        _check(lib.rb_aux_begin(ctx))
        copy(ties if n % 2 else values)
        _check(lib.rb_aux_end(ctx, C.c_uint32(0)))
        RT.token_log_probs(client, x, i, top_k=top, out=out)
        _check(lib.rb_aux_wait(ctx, C.c_uint32(0)))
    client.sync()
    copy(values)
    RT.token_log_probs(client, x, i, top_k=top, out=out)
    compare([client.read(o) for o in out], R.scores(xv, ids, 1.0, -100, top), vocab, top)
    assert not client.read(ties).any() and np.array_equal(client.read(values), xv)
