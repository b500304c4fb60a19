"""GPU: lookups of rows of single bytes (tables held in 8 bits), whose length may be any number of bytes."""
import numpy as np
import pytest

from rust_ascend_b200 import B200Runtime as RT
from rust_ascend_b200 import DType

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("width", [1, 2, 3, 4, 5, 7, 16, 17, 33, 254, 4097])
@pytest.mark.parametrize("values", [np.int8, np.uint8])
@pytest.mark.parametrize("ids", [np.int32, np.int64])
def test_lookup(client, width, values, ids):
    rng = np.random.default_rng(width)
    table = rng.integers(np.iinfo(values).min, np.iinfo(values).max + 1, (37, width)).astype(values)
    at = rng.integers(0, 37, (3, 11)).astype(ids)
    out = RT.embedding(client, client.upload(table), client.upload(at))
    assert out.dtype == (DType.I8 if values is np.int8 else DType.U8)
    assert np.array_equal(client.read(out), table[at])


def test_lookup_in_a_quantised_table(client):
    """A table in 8 bits and its scales, gathered and widened: the rows of the widened table, to the bit."""
    rng = np.random.default_rng(5)
    table = rng.standard_normal((50, 101)).astype(np.float32)
    q, s = RT.quantize_rows(client, client.upload(table))
    ids = client.upload(rng.integers(0, 50, 23))
    s.shape, s.strides = (50, 1), (1, 1)
    rows = RT.embedding(client, q, ids)
    scales = RT.embedding(client, s, ids)
    got = RT.dequantize_rows(client, rows, scales, DType.F32)
    whole = RT.dequantize_rows(client, q, s, DType.F32)
    assert np.array_equal(client.read(got), client.read(whole)[client.read(ids)])
