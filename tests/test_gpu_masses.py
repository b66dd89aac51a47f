"""A step's weights (kv8_mass_dev) against keep_ref.py in 64 bits: calls that attention takes, and what drafted steps leave."""
import copy

import numpy as np
import pytest

import keep_ref as ref
import rehip
from rehip import hip
from test_gpu_attention_sinks import attend_sinks, check_mass, weigh
from test_gpu_kv8 import i32, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("max_rows", [1 << 31, 1 << 40, (1 << 64) - 1])
def test_any_bound_of_the_rows(max_rows):
    """max_rows beyond all rows bounds nothing, as in attention."""
    rng = np.random.default_rng(1)
    bt, cache, q = make(rng, [3, 0, 20], [50, 7, 90], 32, 8, 2, 64)
    check_mass(cache, bt, q, 0.125, 30, 4, max_rows=max_rows, max_len=90)


@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 4)])
@pytest.mark.parametrize("requests", [1, 6, 90])
def test_weights_behind_the_rewind_count_the_rows_that_stay(requests, window, sinks):
    """Behind kv_rewind_dev, with the counts less what went back and the lengths that it left, the weights are those of a step that
    had brought only the rows that stay; the places behind them keep what they had."""
    rng = np.random.default_rng(requests + window)
    page, heads, kv, hd = 32, 8, 2, 64
    rows_of = rng.integers(1, 6, requests)
    bt, cache, q = make(rng, rows_of, rows_of + rng.integers(0, 100, requests), page, heads, kv, hd)
    back = rng.integers(0, rows_of)                               # (the first row stays)
    back[0] = rows_of[0] - 1
    _, lse = attend_sinks(cache, bt, q, 0.125, window, sinks)     # of all rows
    length, free, n_free = i32(bt.len), i32(np.zeros(bt.n_pages)), i32([0])
    rehip.kv_rewind_dev(requests, page, i32(back), length, i32(bt.table), bt.ld, free, bt.n_pages, n_free, length, n_free)
    hip.synchronize()
    stay = copy.copy(bt)
    stay.count, stay.len = (bt.count - back).astype(np.int32), length.download(np.int32, requests)
    np.testing.assert_array_equal(stay.len, bt.len - back)
    start = rng.random(cache.shape[:3]).astype(np.float32)
    want = start.astype(np.float64)
    tol = ref.mass(q, lse, stay.plain(), cache.k, cache.ks, 0.125, window, sinks, want)
    got = weigh(cache, stay, q, lse, 0.125, window, sinks, start, max_rows=5)
    assert np.all(np.abs(got - want) <= tol)
    # rejected rows are not looked at: NaN in their place changes nothing, in weights (to the last bit) and in attention
    q2 = q.copy()
    for b in range(requests):
        q2[bt.start[b] + stay.count[b]:bt.start[b] + bt.count[b]] = np.nan
    _, lse2 = attend_sinks(cache, stay, q2, 0.125, window, sinks, max_rows=5)
    np.testing.assert_array_equal(got, weigh(cache, stay, q2, lse, 0.125, window, sinks, start, max_rows=5))
    live = np.concatenate([np.arange(s, s + c) for s, c in zip(stay.start, stay.count)])
    off = np.abs(lse2[live] - lse[live])
    assert np.all(off <= 2 * ref.attention(q, stay.plain(), (cache.k, cache.v, cache.ks, cache.vs), 0.125, window, sinks,
                                                  np.zeros(q.shape), np.zeros(lse.shape))[1][live])


# (KV heads, rows of the longest, max_len planned for), with 8 query heads of a KV head: a wave for each piece, two (heads beyond 128),
# four waves (many pieces), eight (so many that each has a CU, more than that of half the size) and sixteen
SHARED = {"few rows": (2, 5, 400), "many pieces": (2, 40, 18000), "a round": (2, 40, 4500), "few pieces": (1, 40, 400)}


@pytest.mark.parametrize("name", SHARED)
@pytest.mark.parametrize("hd,page", [(32, 64), (64, 32), (96, 128), (128, 64), (160, 32), (192, 96), (224, 32), (256, 64)])
def test_shares_of_waves_of_every_head_size(name, hd, page):
    kv, rows, max_len = SHARED[name]
    rng = np.random.default_rng(hd + rows)
    bt, cache, q = make(rng, [rows, rows - 3], [300, 77], page, 8 * kv, kv, hd)
    for window, sinks in ((0, 0), (50, 9)):
        check_mass(cache, bt, q, hd ** -0.5, window, sinks, max_rows=rows, max_len=max_len)


@pytest.mark.parametrize("requests", [70, 1030])
@pytest.mark.parametrize("hd,rows", [(64, 3), (128, 1), (192, 1), (256, 2)])
def test_many_requests_of_larger_heads(requests, hd, rows):
    rng = np.random.default_rng(requests + hd)
    rows_of = rng.integers(0, rows + 1, requests)
    bt, cache, q = make(rng, rows_of, rows_of + rng.integers(0, 70, requests), 32, 4, 2, hd)
    check_mass(cache, bt, q, hd ** -0.5, 30, 3)
