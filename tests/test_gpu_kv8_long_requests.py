"""Attention of requests that count more tokens than their table has room for: rows keep their positions, and the tokens
behind the table are not seen, as those of absent pages."""
import numpy as np
import pytest

import serving_ref as ref
from test_gpu_kv8 import attend, make

pytestmark = pytest.mark.gpu


def check(bt, cache, q, scale, window, **k):
    wide = np.full((len(bt.len), int(bt.len.max()) // bt.page + 1), -1, np.int32)
    wide[:, :bt.ld] = bt.table
    want = np.full(q.shape, 7.25)
    tol = ref.attention(q, bt.start, bt.count, bt.len, wide, bt.page, cache.k, cache.v, cache.ks, cache.vs, scale, window,
                        want)
    got = attend(cache, bt, q, scale, window, **k)
    assert np.all(np.abs(got - want) <= tol[..., None]), np.abs(got - want).max()
    return got


@pytest.mark.parametrize("window", [0, 1, 40, 150])
@pytest.mark.parametrize("heads,kv_heads,hd,page,rows_of", [(8, 2, 64, 32, [1, 1, 1, 1, 1]),     # pieces of single rows
                                                            (14, 2, 128, 64, [1, 4, 3, 0, 2]),   # .. of few
                                                            (6, 2, 64, 32, [60, 7, 33, 1, 90]),  # tiles
                                                            (256, 64, 32, 32, [200, 40, 63, 1, 9])])   # wide ones
def test_rows_behind_the_table(heads, kv_heads, hd, page, rows_of, window):
    rng = np.random.default_rng(heads + window)
    room = 6 * page
    bt, cache, q = make(rng, rows_of, [room] * 5, page, heads, kv_heads, hd, gap=1)
    bt.table, bt.ld = np.ascontiguousarray(bt.table[:, :6]), 6
    bt.len[:] = room + 1, room + 5, room, room + 300, room + 60
    got = check(bt, cache, q, hd ** -0.5, window)
    if window == 40 and rows_of[3]:                         # 300 tokens behind: nothing in the window is there
        assert not got[bt.start[3]:bt.start[3] + rows_of[3]].any()


def test_many_requests_behind_their_tables():
    """.. listed pieces, and a wave for each of them"""
    rng = np.random.default_rng(60)
    n = 270
    bt, cache, q = make(rng, np.ones(n, int), np.full(n, 64), 32, 8, 4, 64)
    bt.table, bt.ld = np.ascontiguousarray(bt.table[:, :2]), 2
    bt.len[:] = rng.integers(1, 130, n)
    for max_len in (60, 4000):
        for window in (0, 33):
            check(bt, cache, q, 0.125, window, max_len=max_len)


def test_the_longest_lengths():
    """Positions up to 2^31 - 2: without a window all of the table is seen, with one nothing."""
    rng = np.random.default_rng(61)
    for rows_of in ([1, 3], [50, 1]):
        bt, cache, q = make(rng, rows_of, [128, 128], 64, 8, 2, 64)
        bt.table, bt.ld = np.ascontiguousarray(bt.table[:, :2]), 2
        bt.len[:] = 128 + np.asarray(rows_of)               # (every row sees the whole table)
        want = check(bt, cache, q, 0.125, 0, max_len=200)
        bt.len[:] = 2**31 - 1
        np.testing.assert_array_equal(attend(cache, bt, q, 0.125, max_len=200), want)
        assert not attend(cache, bt, q, 0.125, 1 << 20, max_len=200).any()
