"""Attention with a window and sinks in every form of its launch: tiles of 16, 32 and 64 query vectors of every head size, whole and cut
into pieces, listed, a wave alone, joins of few and of many pieces; eviction's pick by 512 threads. Against keep_ref.py in 64 bits."""
import numpy as np
import pytest

import keep_ref as ref
from test_gpu_attention_sinks import attend_sinks, check, near
from test_gpu_kv8 import make
from test_gpu_kv_evict import check_evict

pytestmark = pytest.mark.gpu
HEAD_SIZES = [(32, 64), (64, 32), (96, 128), (128, 64), (160, 32), (192, 96), (224, 32), (256, 64)]      # and pages
VIEWS = [(0, 0), (50, 9), (20, 40), (200, 33)]


def check_rows(cache, bt, q, scale, window, sinks, rows, **k):
    """As check(), of some rows (of batches that the plain form would take long for)."""
    got, lse = attend_sinks(cache, bt, q, scale, window, sinks, **k)
    want, wl = np.full(q.shape, 7.25), np.full(q.shape[:2], 7.25)
    start, count, kv_len, table, page = bt.plain()
    for r in rows:                       # a request of its own for each
        b = int(np.searchsorted(start, r, "right")) - 1
        p = kv_len[b] - count[b] + r - start[b]
        one = (np.array([r]), np.array([1]), np.array([p + 1]), table[b:b + 1], page)
        tol, tol_lse = ref.attention(q, one, (cache.k, cache.v, cache.ks, cache.vs), scale, window, sinks, want, wl)
        near(got[r], want[r], np.broadcast_to(tol[r][:, None], got[r].shape))
        near(lse[r], wl[r], tol_lse[r])


@pytest.mark.parametrize("rows", [4, 8])
@pytest.mark.parametrize("hd,page", HEAD_SIZES)
def test_wide_tiles_of_few_rows(hd, page, rows):
    """8 heads of a KV head, 4 rows of a request or 8 in tiles of 32 vectors or 64 (up to 128; else several tiles of 32), planned for
    so long requests that tiles are not made smaller to have more of them."""
    rng = np.random.default_rng(hd + rows)
    bt, cache, q = make(rng, [rows, 1, rows, rows - 1], [600, 40, rows, 333], page, 16, 2, hd, gap=1)
    for window, sinks in VIEWS:
        check(cache, bt, q, hd ** -0.5, window, sinks, max_rows=rows, max_len=1 << 20)


@pytest.mark.parametrize("hd,page", HEAD_SIZES)
def test_wide_tiles_of_prompts(hd, page):
    """More than 1024 tiles: 16 KV heads of 4 heads, two prompts."""
    rng = np.random.default_rng(hd)
    n = 1000 if hd <= 128 else 500
    bt, cache, q = make(rng, [n, 90], [n + 130, 200], page, 64, 16, hd)
    some = [0, 1, 15, 16, n // 2, n - 1, n, n + 40, n + 89]
    for window, sinks in VIEWS[1:]:
        check_rows(cache, bt, q, hd ** -0.5, window, sinks, some)


@pytest.mark.parametrize("rows,max_len", [(1, 60), (1, 1 << 16), (4, 1 << 20), (8, 1 << 20)])
@pytest.mark.parametrize("hd,page", HEAD_SIZES)
def test_listed_pieces(hd, page, rows, max_len):
    """More requests than a workgroup looks at: a wave alone where they are short, tiles of 16, 32 and 64 vectors."""
    rng = np.random.default_rng(hd + rows)
    n, heads = 300, 4 if rows == 1 else 8
    rows_of = rng.integers(0, rows + 1, n)
    kv = 4 if rows == 1 else 1
    bt, cache, q = make(rng, rows_of, np.minimum(rows_of + rng.integers(0, 60, n), 60), page, heads, kv, hd)
    some = np.unique(rng.integers(0, bt.rows, 25))
    for window, sinks in ((20, 3), (0, 0)):
        check_rows(cache, bt, q, hd ** -0.5, window, sinks, some, max_rows=rows, max_len=max_len)


@pytest.mark.parametrize("hd,heads", [(32, 1), (64, 5), (128, 2), (256, 1)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (55000, 1024), (30000, 5)])
def test_joins_of_many_pieces(hd, heads, window, sinks):
    """One row over 60000 tokens, cut into a hundred pieces."""
    rng = np.random.default_rng(hd)
    bt, cache, q = make(rng, [1], [60000], 64, heads, 1, hd)
    check(cache, bt, q, hd ** -0.5, window, sinks)


def test_evict_of_requests_between():
    """Up to 8192 tokens: the pick of 512 threads."""
    rng = np.random.default_rng(31)
    check_evict(rng, [5000, 8192, 4097, 300], 64, 2, 32, 4000, 2500, 4, 600, spare=300, masses="fine")
    check_evict(rng, [5000, 8192, 4097, 300], 64, 2, 32, 4000, 2500, 4, 600, spare=300)
