"""GPU: calls of the 8-bit operators and the token scores that their documentation allows and nothing else makes: a recording that forks
to the side stream, inputs whose rows are one and the same, one tensor as both operands, rank one, the last vocabulary entries of split rows."""
import ctypes as C

import numpy as np
import pytest

import eight_bit_reference as R
from rust_ascend_b200 import B200Runtime as RT
from rust_ascend_b200 import DType, TensorBuffer
from rust_ascend_b200.runtime import _check
from test_eight_bit_run_gpu import Block
from test_quant_gpu import NORM_SCALE, SILU, VALUE
from test_scores_gpu import call

pytestmark = pytest.mark.gpu
F32, F16, BF16, I8 = DType.F32, DType.F16, DType.BF16, DType.I8


@pytest.mark.parametrize("sizes", [(40, 300), (3, 3), (600, 1)])
def test_recording_that_forks_to_the_side_stream(client, sizes):
    """One block on each stream, twice, with a fork and a join between: replayed on new inputs, to the bit."""
    a, b = (Block(client, n, 256, 352, 1003, seed=n + i) for i, n in enumerate(sizes))

    def both():
        for _ in range(2):
            _check(client._lib.rb_aux_begin(client._ctx))
            b.run()
            _check(client._lib.rb_aux_end(client._ctx, C.c_uint32(0)))
            a.run()
            _check(client._lib.rb_aux_wait(client._ctx, C.c_uint32(0)))
    a.set(1), b.set(1)
    both()
    client.sync()
    _check(client._lib.rb_graph_begin(client._ctx))
    both()
    g = C.c_uint64()
    _check(client._lib.rb_graph_end(client._ctx, C.byref(g)))
    for seed in (2, 3):
        want = []
        for block in (a, b):
            block.set(seed)
            block.run()
            want.append(block.results())
            for t in (block.q, block.both, block.logits, block.d, *block.scores):
                client.memset(t, 0x55)
        for _ in range(3):
            _check(client._lib.rb_graph_launch(client._ctx, g))
        for block, w in zip((a, b), want):
            for x, y in zip(block.results(), w):
                assert x.tobytes() == y.tobytes()
    _check(client._lib.rb_graph_destroy(client._ctx, g))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("width", [48, 301, 5000])
def test_rows_that_are_one_and_the_same(client, dtype, width):
    """A row distance of zero: every row of the result is that of the one row."""
    rng = np.random.default_rng(width)
    x, xv = R.hold(rng.standard_normal(width), dtype)
    u, uv = R.hold(rng.standard_normal((6, width)), dtype)
    t = client.upload(x, dtype)
    many = TensorBuffer(t.handle, (6, width), dtype, (0, 1), 0, t._owner)
    q, s = RT.quantize_rows(client, many)
    R.check_rows(client.read(q), client.read(s), np.repeat(xv[None].astype(np.float64), 6, 0), 2 * 2.0 ** -24, VALUE)
    q, s = RT.quantize_rows(client, many, up=client.upload(u, dtype))
    R.check_rows(client.read(q), client.read(s), R.silu_mul(np.repeat(xv[None], 6, 0), uv), SILU + 2 * 2.0 ** -24, SILU + VALUE)
    ids = rng.integers(0, width, 6)
    _, out = call(client, None, np.repeat(xv[None], 6, 0), ids, dtype, 1.25, 5, view=many)
    d = RT.token_log_probs_backward(client, many, client.upload(ids), out[1], None, client.upload(np.ones(6, np.float32)), scale=1.25)
    want = R.scores_gradient(np.repeat(xv[None], 6, 0), ids, 1.25, -100, np.ones(6), np.zeros(6))
    # p to 2^-21 and 4 (|z| + |lse|) 2^-24 (both below 16 here), the result to its storage
    assert np.abs(R.read(client, d) - want).max() <= (R.half_step(dtype) + 2.0 ** -16) * 1.25


def test_one_tensor_as_both_operands(client):
    rng = np.random.default_rng(0)
    x, w = rng.standard_normal((9, 304)).astype(np.float32), (1 + 0.1 * rng.standard_normal(304)).astype(np.float32)
    t = client.upload(x)
    q, s, total = RT.rms_norm_quant(client, t, client.upload(w), 1e-5, delta=t)
    assert np.array_equal(client.read(total), x + x)
    R.check_rows(client.read(q), client.read(s), R.norm(x + x, w, 1e-5), NORM_SCALE, VALUE)
    q, s = RT.quantize_rows(client, t, up=t)
    R.check_rows(client.read(q), client.read(s), R.silu_mul(x, x), SILU + 2 * 2.0 ** -24, SILU + VALUE)
    y = client.read(RT.linear_i8(client, q, s, q, s, dtype=F32))
    qv, sv = client.read(q).astype(np.int64), client.read(s)
    assert np.array_equal(y, (qv @ qv.T).astype(np.float32) * (sv[:, None] * sv[None, :]))


def test_rank_one(client):
    rng = np.random.default_rng(0)
    x, w = rng.standard_normal(160).astype(np.float32), np.ones(160, np.float32)
    t = client.upload(x)
    q, s = RT.quantize_rows(client, t)
    assert q.shape == (160,) and s.shape == (1,)
    R.check_rows(client.read(q)[None], client.read(s), x[None].astype(np.float64), 2 * 2.0 ** -24, VALUE)
    q2, s2 = RT.rms_norm_quant(client, t, client.upload(w), 1e-5)
    R.check_rows(client.read(q2)[None], client.read(s2), R.norm(x[None], w, 1e-5), NORM_SCALE, VALUE)
    weight = rng.integers(-127, 128, (37, 160)).astype(np.int8)
    y = RT.linear_i8(client, q, s, client.upload(weight), client.upload(np.ones(37, np.float32)), dtype=F32)
    assert y.shape == (37,)
    assert np.array_equal(client.read(y), (weight.astype(np.int64) @ client.read(q)).astype(np.float32) * client.read(s)[0])
    assert np.array_equal(client.read(RT.dequantize_rows(client, q, s, F32)), client.read(q).astype(np.float32) * client.read(s)[0])
    out = RT.token_log_probs(client, t, client.upload(np.array([7])), top_k=2)
    want = R.scores(x[None], np.array([7]), 1.0, -100, 2)
    assert abs(client.read(out[0])[0] - want[0][0]) <= 2e-6 and np.array_equal(client.read(out[4]).reshape(1, 2), want[4])


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("vocab,pad", [(120001, 1), (99999, 3), (131072, 61)])
@pytest.mark.parametrize("rows,top", [(2, 0), (2, 64), (40, 20)])
def test_few_long_rows_at_any_distance(client, dtype, vocab, pad, rows, top):
    """Rows split over the blocks of a cluster, starting at every distance from a 16-byte boundary, the largest values at the edges of the parts."""
    rng = np.random.default_rng([vocab, rows])
    x, xv = R.hold(rng.standard_normal((rows, vocab + pad)) * 2, dtype)
    edges = [e + o for part in (2, 4, 8) for e in (vocab * i // part for i in range(1, part)) for o in range(-9, 9)] + [0, 1, vocab - 1, vocab - 2]
    big, bv = R.hold(9 + rng.random((rows, len(edges))), dtype)
    x[:, edges], xv[:, edges] = big, bv
    t = client.upload(x, dtype)
    view = TensorBuffer(t.handle, (rows, vocab), dtype, (vocab + pad, 1), 0, t._owner)
    call(client, None, xv[:, :vocab], rng.choice(edges, rows), dtype, 1.0, top, view=view)
