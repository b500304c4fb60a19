"""GPU: how long the sums of token scores get, for rows that are done element by element.

A thread adds at most V / 256 + 16 terms one after the other; test_scores_gpu derives the tolerance from that."""
import numpy as np
import pytest

import eight_bit_reference as R
from rust_ascend_b200 import B200Runtime as RT
from test_scores_gpu import U, compare

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab,top", [(64000, 1), (32768, 0)])
def test_length_of_the_sums_of_rows_done_element_by_element(client, vocab, top):
    """Many rows (blocks of 128 threads) under a scale that sends them there.  Every thread meets a 1 first and then values just below half a step of
    1, which a running sum that holds the 1 loses one by one: as many as there are in it."""
    x = np.full((600, vocab), -16640, np.float16)
    x[:, :128] = 0
    scale = float(np.float32(0.001))
    assert 0.99 * U < np.exp(-16640 * scale) < U
    ids = np.full(600, 5)
    out = RT.token_log_probs(client, client.upload(x), client.upload(ids), scale=scale, top_k=top)
    want = R.scores(x[:1].astype(np.float32), ids[:1], scale, -100, top)
    got = [None if o is None else client.read(o) for o in out]
    compare(got, [np.repeat(w, 600, 0) for w in want], vocab, top)
