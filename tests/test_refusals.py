"""CPU: argument checks of the 8-bit rows, the 8-bit linear and the token scores.  Every call here is refused before anything is
launched, on a context without a device."""
import pytest

from host_context import HostClient
from rust_ascend_b200 import B200Runtime as RT
from rust_ascend_b200 import DType, InvalidTensor, TensorBuffer
from rust_ascend_b200.runtime import NullHandle

F32, F16, BF16, I8, U8, I32, I64 = DType.F32, DType.F16, DType.BF16, DType.I8, DType.U8, DType.I32, DType.I64


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    c = HostClient(str(tmp_path_factory.mktemp("host")))
    yield c
    c.close()


def refused(match, call, *args, **kwargs):
    with pytest.raises(InvalidTensor, match=match):
        call(*args, **kwargs)


def test_norm_quant(host):
    t = host.tensor
    x, w, q, s = t((4, 64), BF16), t((64,), BF16), t((4, 64), I8), t((4,), F32)

    def call(match, x=x, w=w, eps=1e-5, delta=None, out=(q, s)):
        refused(match, RT.rms_norm_quant, host, x, w, eps, delta=delta, out=out)
    call("F32, BF16 or F16", x=t((4, 64), I32))
    call("weight of x's type or F32", w=t((64,), F16))
    call("one value per column", w=t((63,), BF16))
    call("epsilon", eps=0.0)
    call("epsilon", eps=-1.0)
    call("epsilon", eps=float("nan"))
    call("epsilon", eps=1e300)
    call("I8 of the input's shape", out=(t((4, 64), U8), s))
    call("I8 of the input's shape", out=(t((4, 63), I8), s))
    call("one value per row", out=(q, t((5,), F32)))
    call("one value per row", out=(q, t((4,), BF16)))
    call("x's shape and type", delta=t((4, 32), BF16))
    call("x's shape and type", delta=t((4, 64), F32))
    call("come together", out=(q, s, t((4, 64), BF16)))
    call("overlaps", out=(TensorBuffer(x.handle, (4, 64), I8), s))
    call("contiguous", x=TensorBuffer(host.storage(4096), (4, 64), BF16, (128, 1)))
    call("positive last dimension", x=t((4, 0), BF16), w=t((0,), BF16), out=(t((4, 0), I8), s))
    refused("at most 3", RT.rms_norm_quant, host, x, w, 1e-5, out=(q, s, None, None))
    delta = t((4, 64), BF16)
    call("overlaps", delta=delta, out=(q, s, delta))                          # the sum may replace x, not delta


def test_quantize_rows(host):
    t = host.tensor
    x, q, s = t((4, 64), F32), t((4, 64), I8), t((4,), F32)

    def call(match, x=x, up=None, out=(q, s)):
        refused(match, RT.quantize_rows, host, x, up=up, out=out)
    call("F32, BF16 or F16", x=t((4, 64), I64))
    call("one shape and type", up=t((4, 65), F32))
    call("one shape and type", up=t((4, 64), BF16))
    call("last axis must be contiguous", x=TensorBuffer(host.storage(1 << 16), (4, 64), F32, (128, 2)))
    call("at one distance", x=TensorBuffer(host.storage(1 << 20), (2, 2, 64), F32, (1000, 100, 1)), out=(t((2, 2, 64), I8), s))
    call("outside the storage", x=TensorBuffer(host.storage(4 * (3 * 100 + 64) - 1), (4, 64), F32, (100, 1)))
    call("outside the storage", x=TensorBuffer(host.storage(4096), (4, 64), F32, (2**61, 1)))
    call("outside the storage", x=TensorBuffer(host.storage(64), (4, 64), F32, None, 65))
    call("aligned to its element", x=TensorBuffer(host.storage(4096), (4, 64), F32, None, 2))
    call("I8 of the input's shape", out=(t((4, 64), F32), s))
    call("overlaps", out=(TensorBuffer(x.handle, (4, 64), I8), s))
    call("overlaps", out=(q, TensorBuffer(q.handle, (4,), F32)))
    with pytest.raises(NullHandle, match="unknown storage"):
        RT.quantize_rows(host, TensorBuffer(999999, (4, 64), F32), out=(q, s))


def test_dequantize_rows(host):
    t = host.tensor
    q, s, y = t((4, 64), I8), t((4,), F32), t((4, 64), BF16)
    refused("F32, BF16 or F16", RT.dequantize_rows, host, q, s, out=t((4, 64), I32))
    refused("I8 of the input's shape", RT.dequantize_rows, host, t((4, 64), U8), s, out=y)
    refused("one value per row", RT.dequantize_rows, host, q, t((3,), F32), out=y)
    refused("overlaps", RT.dequantize_rows, host, TensorBuffer(y.handle, (4, 64), I8), s, out=y)


def test_linear_i8(host):
    t = host.tensor
    x, sx, w, sw, y = t((5, 64), I8), t((5,), F32), t((48, 64), I8), t((48,), F32), t((5, 48), BF16)

    def call(match, x=x, sx=sx, w=w, sw=sw, bias=None, y=y):
        refused(match, RT.linear_i8, host, x, sx, w, sw, bias=bias, out=y)
    call("I8 operands", x=t((5, 64), U8))
    call("I8 operands", w=t((48, 64), BF16))
    call("must be FP32", sx=t((5,), BF16))
    call("must be FP32", bias=t((48,), BF16))
    call("F32, BF16 or F16", y=t((5, 48), I32))
    call("do not agree", w=t((48, 32), I8))
    call("do not agree", sx=t((4,), F32))
    call("do not agree", sw=t((47,), F32))
    call("do not agree", bias=t((47,), F32))
    call("do not agree", y=t((4, 48), BF16))
    call("do not agree", x=t((5, 1, 64), I8), y=t((1, 5, 48), BF16))
    call("multiple of 16", x=t((5, 40), I8), w=t((48, 40), I8))
    call("within 131056", x=t((5, 131072), I8), w=t((48, 131072), I8))
    call("overlaps", y=TensorBuffer(w.handle, (5, 48), BF16))
    call("16-byte aligned", x=TensorBuffer(host.storage(4096, misalign=8), (5, 64), I8))
    call(r"X\[..,K\] and W\[N,K\]", w=t((1, 48, 64), I8))
    call("N must be positive", w=t((0, 64), I8), sw=t((0,), F32), y=t((5, 0), BF16))


def test_token_log_probs(host):
    t = host.tensor
    logits, ids = t((3, 100), F32), t((3,), I64)
    out = [t((3,), F32) for _ in range(3)]

    def call(match, logits=logits, ids=ids, scale=1.0, top=0, out=out):
        refused(match, RT.token_log_probs, host, logits, ids, scale=scale, top_k=top, out=out)
    call("F32, BF16 or F16", logits=t((3, 100), I32))
    call("INT32 or INT64", ids=t((3,), F32))
    call("one id per row", ids=t((4,), I64))
    call("positive and finite", scale=0.0)
    call("positive and finite", scale=-1.0)
    call("positive and finite", scale=float("inf"))
    call("positive and finite", scale=float("nan"))
    call("within 0..64", top=65, out=out + [t((3, 65), F32), t((3, 65), I32)])
    call("within 0..64", top=-1)
    call("and the vocabulary", logits=t((3, 10), F32), top=11, out=out + [t((3, 11), F32), t((3, 11), I32)])
    call("come with a positive top_k", top=2)
    call("come with a positive top_k", out=out + [t((3, 2), F32), t((3, 2), I32)])
    call("top_ids must be I32", top=2, out=out + [t((3, 2), F32), t((3, 2), I64)])
    call("lse must be F32", out=[out[0], t((4,), F32), out[2]])
    call("missing tensor", out=[None, out[1], out[2]])
    call("overlaps", out=[out[0], out[0], out[2]])
    call("overlaps", out=[TensorBuffer(logits.handle, (3,), F32), out[1], out[2]])
    call("outside the storage", logits=TensorBuffer(host.storage(1000), (3, 100), F32, (101, 1)))


def test_token_log_probs_backward(host):
    t = host.tensor
    logits, ids, row = t((3, 100), BF16), t((3,), I32), [t((3,), F32) for _ in range(4)]
    d = t((3, 100), BF16)

    def call(match, logits=logits, ids=ids, lse=row[0], entropy=row[1], g=row[2], h=row[3], out=d):
        refused(match, RT.token_log_probs_backward, host, logits, ids, lse, entropy, g, h, out=out)
    call("needs the saved entropy", entropy=None)
    call("shape and type", out=t((3, 100), F32))
    call("shape and type", out=t((3, 99), BF16))
    call("grad_log_probs must be F32", g=t((2,), F32))
    call("lse must be F32", lse=t((3,), I32))
    call("overlap", out=TensorBuffer(host.storage(4096), (3, 100), BF16, (50, 1)))
    wide = host.storage(4096)
    call("overlaps", logits=TensorBuffer(wide, (3, 100), BF16, (200, 1)), out=TensorBuffer(wide, (3, 100), BF16, (200, 1), 200))   # a shifted view of the logits
    call("overlaps", lse=TensorBuffer(d.handle, (3,), F32))


def test_empty_batches_return_without_a_launch(host):
    t = host.tensor
    before = host.stats()
    RT.rms_norm_quant(host, t((0, 64), F32), t((64,), F32), 1e-5, out=(t((0, 64), I8), t((0,), F32)))
    RT.quantize_rows(host, t((0, 64), F32), out=(t((0, 64), I8), t((0,), F32)))
    RT.dequantize_rows(host, t((0, 64), I8), t((0,), F32), out=t((0, 64), F32))
    RT.linear_i8(host, t((0, 64), I8), t((0,), F32), t((48, 64), I8), t((48,), F32), out=t((0, 48), F32))
    RT.token_log_probs(host, t((0, 64), F32), t((0,), I32), out=[t((0,), F32) for _ in range(3)])
    RT.token_log_probs_backward(host, t((0, 64), F32), t((0,), I32), t((0,), F32), None, t((0,), F32), out=t((0, 64), F32))
    after = host.stats()
    assert after["empty_calls"] == before["empty_calls"] + 6 and after["launches"] == before["launches"]


def test_column_ranges_of_an_empty_batch(host):
    """A range of the columns of a tensor without rows starts behind its storage, which nothing reads."""
    t = host.tensor
    both = t((0, 128), BF16)
    half = lambda at: TensorBuffer(both.handle, (0, 64), BF16, (128, 1), both.offset + at * 2)
    before = host.stats()
    RT.quantize_rows(host, half(0), up=half(64), out=(t((0, 64), I8), t((0,), F32)))
    RT.token_log_probs(host, half(64), t((0,), I32), out=[t((0,), F32) for _ in range(3)])
    assert host.stats()["empty_calls"] == before["empty_calls"] + 2
    refused("outside the storage", RT.quantize_rows, host, TensorBuffer(both.handle, (1, 64), BF16, None, 128), out=(t((1, 64), I8), t((1,), F32)))


def test_swiglu_shapes(host):
    from rust_ascend_b200 import nn
    pair = lambda n, k: nn.QuantizedRows(nn.Tensor(host, host.tensor((n, k), I8)), nn.Tensor(host, host.tensor((n,), F32)))
    flat = nn.QuantizedRows(nn.Tensor(host, host.tensor((64,), I8)), nn.Tensor(host, host.tensor((1,), F32)))
    for x, gate_up, down in ((flat, pair(96, 64), pair(32, 48)), (pair(4, 64), pair(95, 64), pair(32, 48)), (pair(4, 64), flat, pair(32, 48)), (pair(4, 64), pair(96, 64), flat)):
        refused("SwiGLU", nn.swiglu_quantized, x, gate_up, down)


def test_descriptor_follows_the_fields():
    """The C descriptor of a tensor is made once and dropped when a field changes."""
    import copy
    from rust_ascend_b200.runtime import _ref
    t = TensorBuffer(3, (2, 8), F32)
    first = _ref(t)
    assert _ref(t) is first and list(first._obj.shape[:2]) == [2, 8]
    t.shape, t.strides = (4, 4), (4, 1)
    d = _ref(t)._obj
    assert (d.rank, list(d.shape[:2]), list(d.strides[:2])) == (2, [4, 4], [4, 1])
    other = copy.deepcopy(t)
    other.offset = 16
    assert _ref(other)._obj.offset == 16 and _ref(t)._obj.offset == 0 and other != t
