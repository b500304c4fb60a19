"""GPU: token scores and their gradient at both ends of what the scale may be.

Tolerances are those of test_scores_gpu.  At the ends an exponent has four roundings instead of three (difference, scale, product with
log2 e or its double, and that constant), but the vocabularies here are below 2^12, so its weighted size is below 12 and 4 x 12 < 3 x 17."""
import numpy as np
import pytest

import eight_bit_reference as R
from rust_ascend_b200 import B200Runtime as RT
from rust_ascend_b200 import DType
from test_scores_gpu import U, call, gradient_error

pytestmark = pytest.mark.gpu
F32, F16, BF16 = DType.F32, DType.F16, DType.BF16
LARGEST = float(np.finfo(np.float32).max)


def rows_at(scale, dtype, spread, rows=5, vocab=3001):
    """Logits whose product with the scale is about `spread`, one row with masks, and ids."""
    rng = np.random.default_rng([int(-np.log10(spread) * 10) + 1000, int(dtype)])
    x, xv = R.hold(np.clip(rng.standard_normal((rows, vocab)) * spread / scale, -3.3e38, 3.3e38), dtype)
    minus = {F32: np.float32(-np.inf), BF16: np.uint16(0xff80), F16: np.float16(-np.inf)}[dtype]
    x, xv = x.copy(), xv.copy()
    x[1, 100:], xv[1, 100:] = minus, -np.inf
    ids = rng.integers(0, vocab, rows)
    ids[1], ids[2] = 7, -100
    return rng, x, xv, ids


# 2.4e38 log2 e is beyond FP32; 1e-38 times logits that lie more than FP32's largest value apart; 1e-41 is denormal
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("scale", [1e-41, 1e-38, 2.3e38, 2.4e38, LARGEST])
@pytest.mark.parametrize("top", [0, 6])
def test_scales_at_the_ends(client, dtype, scale, top):
    scale = float(np.float32(scale))
    _, x, xv, ids = rows_at(scale, dtype, min(2.5, 1.1e38 * scale))
    call(client, x, xv, ids, dtype, scale, top)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("scale", [2.4e38, LARGEST])
def test_certain_rows_under_the_largest_scales(client, dtype, scale):
    """Ordinary logits: the largest takes all, and lse may be beyond FP32's range."""
    rng = np.random.default_rng(1)
    x, xv = R.hold(rng.standard_normal((4, 701)) * [[0.2], [0.05], [1], [3]], dtype)
    call(client, x, xv, np.array([3, int(xv[1].argmax()), -100, 700]), dtype, float(np.float32(scale)), 4)


@pytest.mark.parametrize("dtype,scale", [(F32, 1e-41), (F32, 1e-38), (BF16, 1e-38), (F32, 2.4e38), (BF16, 2.4e38), (F32, LARGEST), (BF16, LARGEST)])
@pytest.mark.parametrize("out", ["same", "shifted"])
def test_gradient_at_the_ends(client, dtype, scale, out):
    scale = float(np.float32(scale))
    rng, x, xv, ids = rows_at(scale, dtype, min(2.5, 1.1e38 * scale))
    rows, vocab = x.shape
    g, h = (0.2 * rng.standard_normal(rows)).astype(np.float32), (0.02 * rng.standard_normal(rows)).astype(np.float32)
    t, s = call(client, x, xv, ids, dtype, scale, 0)
    d = client.tensor((rows, vocab), dtype)
    if out == "shifted":
        wide = client.tensor((rows, vocab + 3), dtype)
        d = type(wide)(wide.handle, (rows, vocab), dtype, (vocab + 3, 1), dtype.size, wide._owner)
        client.memset(wide, 0)
    RT.token_log_probs_backward(client, t, client.upload(ids), s[1], s[2], client.upload(g), client.upload(h), scale=scale, out=d)
    got = R.read(client, d) if out == "same" else R.read(client, wide)[:, 1:vocab + 1]
    want = R.scores_gradient(xv, ids, scale, -100, g, h)
    assert np.abs(want).max() < LARGEST
    half = R.half_step(dtype)
    smallest = {F32: 2.0 ** -149, BF16: 2.0 ** -133}[dtype]
    off = np.abs(got.astype(np.float64) - want) - (gradient_error(xv, ids, scale, g, h, dtype) * (1 + half) + (half + 6 * U) * np.abs(want) + smallest)
    assert off.max() <= 0, (off.max(), np.isnan(got).any())
    assert not got[1, 100:].any()


@pytest.mark.parametrize("dtype,scale", [(F16, 1e-30), (F16, 1e-3), (F16, 0.014), (F16, 0.02), (BF16, 1e-35), (BF16, 1e-37), (F32, 1e-34), (F32, 1e-36)])
@pytest.mark.parametrize("with_entropy", [False, True])
@pytest.mark.parametrize("upstream", [1.0, 1e30])
def test_gradient_on_both_sides_of_the_scale_that_goes_element_by_element(client, dtype, scale, with_entropy, upstream):
    """Nearly uniform rows under scales at which the masks' stand-in no longer fits the type, and just above; gradients of order one, or large ones of the scores."""
    scale = float(np.float32(scale))
    rng = np.random.default_rng([int(-np.log10(scale)), int(dtype)])
    rows, vocab = 5, 1003
    x, xv = R.hold(np.clip(rng.standard_normal((rows, vocab)) * min(3 / scale, 60000 if dtype == F16 else 1e38) / 4, -65504 if dtype == F16 else -3e38, 65504 if dtype == F16 else 3e38), dtype)
    ids = rng.integers(0, vocab, rows)
    ids[3] = -100
    size = min(upstream, 0.1 / scale)
    g, h = (size * rng.standard_normal(rows)).astype(np.float32), (size * 0.3 * rng.standard_normal(rows)).astype(np.float32) * with_entropy
    t, s = call(client, x, xv, ids, dtype, scale, 0)
    up = client.upload
    d = RT.token_log_probs_backward(client, t, up(ids), s[1], s[2] if with_entropy else None, up(g), up(h) if with_entropy else None, scale=scale)
    got, want = R.read(client, d).astype(np.float64), R.scores_gradient(xv, ids, scale, -100, g, h)
    half = R.half_step(dtype)
    smallest = {F32: 2.0 ** -149, BF16: 2.0 ** -133, F16: 2.0 ** -24}[dtype]
    off = np.abs(got - want) - (gradient_error(xv, ids, scale, g, h, dtype) * (1 + half) + (half + 6 * U) * np.abs(want) + smallest)
    assert off.max() <= 0, off.max()
