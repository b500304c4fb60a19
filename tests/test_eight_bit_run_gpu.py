"""GPU: the 8-bit operators and the token scores run together: a feed-forward block and a language-model head in 8 bits up to the scores
and their gradient, eagerly, recorded into a graph, and on the side stream."""
import ctypes as C

import numpy as np
import pytest

import eight_bit_reference as R
from rust_ascend_b200 import B200Runtime as RT
from rust_ascend_b200 import DType, TensorBuffer
from rust_ascend_b200.runtime import _check

pytestmark = pytest.mark.gpu
F32, BF16, I8, I32 = DType.F32, DType.BF16, DType.I8, DType.I32


class Block:
    """Weights held in 8 bits, and every intermediate tensor allocated once, as a serving loop keeps them."""

    def __init__(self, client, tokens, hidden, ffn, vocab, seed=0):
        self.c, self.tokens, self.ffn, self.vocab = client, tokens, ffn, vocab
        rng = np.random.default_rng(seed)
        up = client.upload

        def weight(n, k):
            v = (rng.standard_normal((n, k)) / np.sqrt(k)).astype(np.float32)
            q, s = RT.quantize_rows(client, up(v))
            return q, s, client.read(q).astype(np.float64) * client.read(s).astype(np.float64)[:, None]
        self.gate_up, self.down, self.head = weight(2 * ffn, hidden), weight(hidden, ffn), weight(vocab, hidden)
        self.norm_w = [R.hold(1 + 0.1 * rng.standard_normal(hidden), BF16) for _ in range(2)]
        self.w = [up(b, BF16) for b, _ in self.norm_w]
        t = client.tensor
        self.x, self.q, self.s = t((tokens, hidden), BF16), t((tokens, hidden), I8), t((tokens,), F32)
        self.both, self.hq, self.hs = t((tokens, 2 * ffn), BF16), t((tokens, ffn), I8), t((tokens,), F32)
        self.delta, self.total, self.q2, self.s2 = t((tokens, hidden), BF16), t((tokens, hidden), BF16), t((tokens, hidden), I8), t((tokens,), F32)
        self.logits, self.ids = t((tokens, vocab), BF16), t((tokens,), I32)
        self.scores = [t((tokens,), F32) for _ in range(3)] + [t((tokens, 5), F32), t((tokens, 5), I32)]
        self.g, self.d = t((tokens,), F32), t((tokens, vocab), BF16)

    def set(self, seed):
        rng = np.random.default_rng(seed)
        self.x_bits, self.x_values = R.hold(rng.standard_normal((self.tokens, self.x.shape[1])), BF16)
        self.id_values = rng.integers(0, self.vocab, self.tokens).astype(np.int32)
        self.g_values = rng.standard_normal(self.tokens).astype(np.float32)
        for t, a in ((self.x, self.x_bits), (self.ids, self.id_values), (self.g, self.g_values)):
            self.c.write(t.handle, np.ascontiguousarray(a))
        self.c.sync()

    def run(self):
        c, f = self.c, self.ffn
        RT.rms_norm_quant(c, self.x, self.w[0], 1e-5, out=(self.q, self.s))
        RT.linear_i8(c, self.q, self.s, *self.gate_up[:2], out=self.both)
        gate = TensorBuffer(self.both.handle, (self.tokens, f), BF16, (2 * f, 1))
        up = TensorBuffer(self.both.handle, (self.tokens, f), BF16, (2 * f, 1), 2 * f)
        RT.quantize_rows(c, gate, up=up, out=(self.hq, self.hs))
        RT.linear_i8(c, self.hq, self.hs, *self.down[:2], out=self.delta)
        RT.rms_norm_quant(c, self.x, self.w[1], 1e-5, delta=self.delta, out=(self.q2, self.s2, self.total))
        RT.linear_i8(c, self.q2, self.s2, *self.head[:2], out=self.logits)
        RT.token_log_probs(c, self.logits, self.ids, top_k=5, out=self.scores)
        RT.token_log_probs_backward(c, self.logits, self.ids, self.scores[1], self.scores[2], self.g, self.g, out=self.d)

    def results(self):
        return [self.c.read(t) for t in (self.q, self.both, self.hq, self.delta, self.total, self.q2, self.logits, *self.scores, self.d)]

    def in_64_bits(self):
        def held(y):
            s = R.scale_of(y)[:, None]
            return np.rint(y / s) * s
        h = held(R.norm(self.x_values, self.norm_w[0][1], 1e-5))
        both = h @ self.gate_up[2].T
        h = held(R.silu_mul(both[:, :self.ffn], both[:, self.ffn:]))
        total = self.x_values + h @ self.down[2].T
        return total, held(R.norm(total, self.norm_w[1][1], 1e-5)) @ self.head[2].T


@pytest.mark.parametrize("tokens", [1, 5, 130, 700])
def test_block(client, tokens):
    b = Block(client, tokens, 256, 352, 1003)
    b.set(1)
    b.run()
    total, logits = b.in_64_bits()
    # Activations are rounded to BF16 between the operators and once to 8 bits after each: values of order one that differ by half a BF16
    # step move an 8-bit value by one step now and then, so the comparison is of the whole, not of single elements.
    got = R.read(client, b.total)
    assert np.linalg.norm(got - total) <= 0.01 * np.linalg.norm(total)
    x = R.read(client, b.logits)
    assert np.linalg.norm(x - logits) <= 0.03 * np.linalg.norm(logits)
    # the scores are exact functions of the logits that are there
    want = R.scores(x, b.id_values, 1.0, -100, 5)
    for t, w in zip(b.scores[:4], want[:4]):
        assert np.abs(client.read(t) - w).max() <= 2e-5
    assert np.array_equal(client.read(b.scores[4]), want[4])
    d = R.scores_gradient(x, b.id_values, 1.0, -100, b.g_values, b.g_values)
    assert np.abs(R.read(client, b.d) - d).max() <= 2.0 ** -8 * np.abs(d).max()


@pytest.mark.parametrize("tokens", [3, 600])
def test_recorded_and_replayed_on_new_inputs(client, tokens):
    """One recording of the whole run, replayed on other inputs, gives what eager calls give: to the bit, since no result depends on an
    order of additions that could change.  Two recordings replayed one after the other share nothing."""
    blocks = [Block(client, tokens, 256, 352, 1003, seed=s) for s in range(2)]
    graphs = []
    for b in blocks:
        b.set(1)
        b.run()                                       # first use configures the kernels
        client.sync()
        _check(client._lib.rb_graph_begin(client._ctx))
        b.run()
        g = C.c_uint64()
        _check(client._lib.rb_graph_end(client._ctx, C.byref(g)))
        graphs.append(g)
    for seed in (2, 3):
        eager = []
        for b in blocks:
            b.set(seed)
            b.run()
            eager.append(b.results())
            for t in (b.q, b.both, b.logits, b.d, *b.scores):
                client.memset(t, 0x55)
        for g in graphs:
            _check(client._lib.rb_graph_launch(client._ctx, g))
        for b, want in zip(blocks, eager):
            for a, w in zip(b.results(), want):
                assert a.tobytes() == w.tobytes()
    for g in graphs:
        _check(client._lib.rb_graph_destroy(client._ctx, g))


def test_side_stream_beside_the_compute_stream(client):
    """Two blocks at once, one on the compute stream, one on the side stream."""
    a, b = Block(client, 40, 256, 352, 1003, seed=4), Block(client, 300, 256, 352, 1003, seed=5)
    a.set(6), b.set(7)
    a.run(), b.run()
    want = [a.results(), b.results()]
    for t in (a.logits, a.d, b.logits, b.d):
        client.memset(t, 0x55)
    for _ in range(3):
        _check(client._lib.rb_aux_begin(client._ctx))
        b.run()
        _check(client._lib.rb_aux_end(client._ctx, C.c_uint32(0)))
        a.run()
        _check(client._lib.rb_aux_wait(client._ctx, C.c_uint32(0)))
    for block, w in zip((a, b), want):
        for x, y in zip(block.results(), w):
            assert x.tobytes() == y.tobytes()


def test_calls_from_another_thread(client):
    """The entry points make the context's device current themselves, and take calls from any thread."""
    import threading
    b = Block(client, 17, 256, 352, 1003, seed=9)
    b.set(1)
    b.run()
    want = b.results()
    failed = []

    def work():
        try:
            b.run()
            client.sync()
        except Exception as e:                       # reported by the assertion below
            failed.append(e)
    t = threading.Thread(target=work)
    t.start()
    t.join()
    assert not failed
    for x, y in zip(b.results(), want):
        assert x.tobytes() == y.tobytes()


def test_steady_state_allocates_nothing(client):
    b = Block(client, 9, 256, 352, 1003, seed=2)
    b.set(1)
    b.run()
    before = client.stats()
    for _ in range(5):
        b.run()
    client.sync()
    after = client.stats()
    assert after["allocations"] == before["allocations"] and after["bytes_in_use"] == before["bytes_in_use"]
    assert after["launches"] - before["launches"] == 5 * 8


def test_nn_functions(client):
    """The tensor-level functions: a feed-forward block, its norm, and the scores of its result."""
    from rust_ascend_b200 import InvalidTensor, nn
    rng = np.random.default_rng(12)
    T = lambda a, dtype=None: nn.Tensor.from_data(client, a, dtype)
    (xb, xv), (db, dv), (wb, wv) = (R.hold(rng.standard_normal(s), BF16) for s in ((33, 256), (33, 256), (256,)))
    gate_up, down = ((rng.standard_normal(s) / np.sqrt(s[1])).astype(np.float32) for s in ((2 * 352, 256), (256, 352)))
    total, q = nn.add_rms_norm_quantized(T(xb, BF16), T(db, BF16), T(wb, BF16), 1e-5)
    alone = nn.rms_norm_quantized(total, T(wb, BF16), 1e-5)
    assert np.array_equal(alone.values.into_data(), q.values.into_data()) and np.array_equal(alone.scales.into_data(), q.scales.into_data())
    wg, wd = nn.quantize_rows(T(gate_up)), nn.quantize_rows(T(down))
    y = nn.swiglu_quantized(q, wg, wd, F32)
    h = q.dequantize().into_data().astype(np.float64)
    both = R.hold(h @ wg.dequantize().into_data().astype(np.float64).T, BF16)[1]
    act = nn.silu_mul_quantized(T(R.hold(both[:, :352], BF16)[0], BF16), T(R.hold(both[:, 352:], BF16)[0], BF16)).dequantize().into_data().astype(np.float64)
    want = act @ wd.dequantize().into_data().astype(np.float64).T
    assert np.linalg.norm(y.into_data() - want) <= 0.01 * np.linalg.norm(want)         # a BF16 rounding of `both` may fall on the other side
    logits, ids = T((rng.standard_normal((33, 1003)) * 2).astype(np.float32)), T(rng.integers(0, 1003, 33))
    s = nn.TokenScoreConfig(temperature=0.8, alternatives=3).forward(logits, ids)
    w = R.scores(logits.into_data(), ids.into_data(), np.float32(1 / 0.8), -100, 3)
    for a, b in zip((s.log_probs, s.lse, s.entropy, s.top_log_probs), w):
        assert np.abs(a.into_data() - b).max() <= 2e-5
    assert np.array_equal(s.top_ids.into_data(), w[4])
    g = np.ones(33, np.float32)
    d = s.backward(T(g), T(g)).into_data()
    assert np.abs(d - R.scores_gradient(logits.into_data(), ids.into_data(), np.float32(1 / 0.8), -100, g, g)).max() <= 1e-5
    assert nn.TokenScoreConfig().forward(logits, ids).top_ids is None
    with pytest.raises(InvalidTensor, match="temperature"):
        nn.TokenScoreConfig(temperature=0.0).forward(logits, ids)
    with pytest.raises(InvalidTensor, match="SwiGLU"):
        nn.swiglu_quantized(q, wd, wg)


def test_every_operand_from_the_kernel_in_front(client):
    """Activations, scales, weights of the norm and of the linear, logits and saved statistics: each rewritten by the call right in front of
    the one that reads it, after an earlier call has read the same addresses.  The results are those of calls that wait for each other."""
    rng = np.random.default_rng(21)
    rows, k, n = 3, 1024, 640                              # 3 tokens: the linear that reads its operands with ordinary loads
    t = client.tensor
    source = [client.upload((rng.standard_normal((n, k)) * (1 + i)).astype(np.float32)) for i in range(4)]
    x = t((rows, k), F32)
    w8, ws, xq, xs, nq, ns = t((n, k), I8), t((n,), F32), t((rows, k), I8), t((rows,), F32), t((1, k), I8), t((1,), F32)
    weight, y = t((k,), F32), t((rows, n), F32)
    ids = client.upload(rng.integers(0, n, rows))
    scores, g, d = [t((rows,), F32) for _ in range(3)], client.upload(np.ones(rows, np.float32)), t((rows, n), F32)
    part = lambda b, first, m: TensorBuffer(b.handle, (m, k), F32, None, first * k * 4, b._owner)

    def round_of(i, wait):
        out = []
        done = client.sync if wait else lambda: None
        s = source[i % 4]
        RT.quantize_rows(client, part(s, 7, 1), out=(nq, ns)); done()
        RT.dequantize_rows(client, nq, ns, out=TensorBuffer(weight.handle, (1, k), F32)); done()
        RT.rms_norm_quant(client, part(s, 8, rows), weight, 1e-5, out=(xq, xs)); done()             # weight from the call in front
        RT.dequantize_rows(client, xq, xs, out=x); done()
        RT.quantize_rows(client, s, out=(w8, ws)); done()
        RT.linear_i8(client, xq, xs, w8, ws, out=y); done()                                         # W and its scales too
        RT.quantize_rows(client, x, out=(xq, xs)); done()
        RT.linear_i8(client, xq, xs, w8, ws, out=y); done()                                         # x and its scales
        RT.token_log_probs(client, y, ids, out=[*scores, None, None]); done()
        RT.token_log_probs_backward(client, y, ids, scores[1], scores[2], g, g, out=d); done()
        RT.rms_norm_quant(client, x, weight, 1e-5, delta=part(s, 30, rows), out=(xq, xs, x)); done()
        for a in (xq, xs, x, y, d, weight):
            copy = t(a.shape, a.dtype)
            _check(client._lib.rb_copy(client._ctx, C.byref(a._c()), C.byref(copy._c())))
            out.append(copy)
        return out
    want = [[client.read(a) for a in round_of(i, True)] for i in range(4)]
    got = [round_of(i, False) for i in range(40)]
    client.sync()
    for i, out in enumerate(got):
        for a, b in zip(out, want[i % 4]):
            assert np.array_equal(client.read(a), b)


def test_copies_and_other_kernels_between(client):
    """The operators start their blocks early behind each other; behind a copy, a fill or a kernel that does not take part they still see its
    result, eagerly and in a recording."""
    rng = np.random.default_rng(3)
    rows, width = 64, 2048
    src, x, y = (client.tensor((rows, width), F32) for _ in range(3))
    q, s, back = client.tensor((rows, width), I8), client.tensor((rows,), F32), client.tensor((rows, width), F32)

    def sequence():
        _check(client._lib.rb_copy(client._ctx, C.byref(src._c()), C.byref(x._c())))
        RT.quantize_rows(client, x, out=(q, s))
        RT.dequantize_rows(client, q, s, out=back)
        RT.add(client, back, x, out=y)                    # an ordinary launch
        RT.quantize_rows(client, y, out=(q, s))
        client.memset(back, 0)
        RT.dequantize_rows(client, q, s, out=back)

    def expected(v):
        def held(a):
            scale = np.maximum(np.abs(a).max(-1, keepdims=True) / np.float32(127), np.float32(R.SMALLEST))
            return np.rint(a.astype(np.float64) / scale) * scale
        return held((held(v).astype(np.float32) + v))
    sequence()
    client.sync()
    _check(client._lib.rb_graph_begin(client._ctx))
    sequence()
    g = C.c_uint64()
    _check(client._lib.rb_graph_end(client._ctx, C.byref(g)))
    for i in range(6):
        v = rng.standard_normal((rows, width)).astype(np.float32) * (i + 1)
        client.write(src.handle, v)
        if i % 2:
            _check(client._lib.rb_graph_launch(client._ctx, g))
        else:
            sequence()
        # a value on the border between two steps may fall on either side: one step of the row's scale
        assert np.abs(client.read(back) - expected(v)).max() <= 1.01 * np.abs(2 * v).max() / 127
        assert np.mean(np.abs(client.read(back) - expected(v)) > 1e-4) < 1e-3
    _check(client._lib.rb_graph_destroy(client._ctx, g))
