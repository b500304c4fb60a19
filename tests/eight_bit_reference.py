"""Definitions in 64 bits of the 8-bit rows, the 8-bit linear and the token scores, for the tests."""
import numpy as np

from rust_ascend_b200 import DType
from rust_ascend_b200.runtime import bf16_bits_to_f32, f32_to_bf16_bits

SMALLEST = 2.0 ** -126


def hold(a, dtype):
    """(host carrier, FP32 values) of an array held in `dtype`."""
    a = np.asarray(a, np.float32)
    if dtype == DType.BF16:
        bits = f32_to_bf16_bits(a)
        return bits, bf16_bits_to_f32(bits)
    if dtype == DType.F16:
        h = a.astype(np.float16)
        return h, h.astype(np.float32)
    return a, a


def read(client, t):
    a = client.read(t)
    return bf16_bits_to_f32(a) if t.dtype == DType.BF16 else a.astype(np.float32) if t.dtype == DType.F16 else a


def half_step(dtype):
    return {DType.F32: 2.0 ** -24, DType.BF16: 2.0 ** -8, DType.F16: 2.0 ** -11}[dtype]


def norm(x, w, eps):
    x = x.astype(np.float64)
    return x * w.astype(np.float64) / np.sqrt((x * x).mean(-1, keepdims=True) + eps)


def silu_mul(g, u):
    g = g.astype(np.float64)
    return g / (1 + np.exp(-g)) * u.astype(np.float64)


def scale_of(y):
    return np.maximum(np.abs(y).max(-1) / 127, SMALLEST)


def check_rows(q, scales, y, scale_error, value_error):
    """q and scales against y in 64 bits: the scale to a relative error, q within half a step plus what y's own relative error moves it."""
    want = scale_of(y)
    assert np.abs(scales / want - 1).max() <= scale_error, np.abs(scales / want - 1).max()
    assert np.abs(q.astype(np.int64)).max() <= 127
    off = np.abs(q - y / want[..., None])
    slack = 127 * value_error
    assert off.max() <= 0.5 + slack, off.max() - 0.5


def scores(x, ids, scale, ignore, top):
    """lp of the ids, lse, entropy, top values and ids of rows of logits (ids outside the vocabulary count as ignored)."""
    z = x.astype(np.float64) * scale
    m = z.max(-1, keepdims=True)
    with np.errstate(all="ignore"):
        lse = np.where(m[:, 0] == -np.inf, -np.inf, m[:, 0] + np.log(np.exp(z - m).sum(-1)))      # log of an empty sum
        lp = (z - m) - np.log(np.exp(z - m).sum(-1, keepdims=True))
        p = np.exp(lp)
        entropy = -np.where(p > 0, p * np.where(p > 0, lp, 0), np.where(np.isnan(p), np.nan, 0)).sum(-1)
    rows, vocab = x.shape
    live = (ids != ignore) & (ids >= 0) & (ids < vocab)
    chosen = np.where(live, lp[np.arange(rows), np.where(live, ids, 0)], 0.0)
    key = np.where(np.isnan(x), np.inf, x.astype(np.float64))
    order = np.lexsort((np.broadcast_to(np.arange(vocab), x.shape), -key, ~np.isnan(x)), axis=-1)[:, :top]
    return chosen, lse, entropy, np.take_along_axis(lp, order, -1), order, live


def scores_gradient(x, ids, scale, ignore, g, h):
    """The formula of the gradient in 64 bits."""
    _, lse, entropy, _, _, live = scores(x, ids, scale, ignore, 0)
    z = x.astype(np.float64) * scale
    lp = z - lse[:, None]
    p = np.exp(lp)
    assert np.all(np.abs(lse) < 1e6)             # beyond it z - lse is not what the formula means, even here
    hot = np.zeros_like(p)
    hot[np.flatnonzero(live), ids[live]] = 1
    plogp = np.where(p > 0, p * np.where(p > 0, lp, 0), 0)
    return scale * (np.where(live, g, 0)[:, None] * (hot - p) - h[:, None] * (plogp + p * entropy[:, None]))
