"""Attention over int8 pages with a sliding window and sinks, and the weights of a step, against the plain restatements of
keep_ref.py: ragged batches, part-filled and absent pages, windows that meet the sinks or not, rows that see nothing."""
import numpy as np
import pytest

import keep_ref as ref
import rehip
from rehip import hip
from test_gpu_kv8 import Batch, Cache, attend, i32, make

pytestmark = pytest.mark.gpu
B = hip.DeviceBuffer


def work_for(rows, bt, max_rows, max_len, heads, kv_heads, hd):
    nb = rehip.attention_kv8_work_bytes(rows, len(bt.count), max(max_rows, 1), max_len, heads, kv_heads, hd)
    return B.from_array(np.full(max(nb // 4, 4), np.nan, np.float32)), nb


def attend_sinks(cache, bt, q, scale, window, sinks, max_rows=None, max_len=None, stream=None, ldq=None, lse=True):
    rows, heads, hd = q.shape
    kv_heads = cache.shape[1]
    ldq = ldq or heads * hd
    full = np.full((rows, ldq), np.nan, np.float32)
    full[:, :heads * hd] = q.reshape(rows, -1)
    max_rows = int(bt.count.max()) if max_rows is None else max_rows
    max_len = int(bt.len.max()) if max_len is None else max_len
    work, nb = work_for(rows, bt, max_rows, max_len, heads, kv_heads, hd)
    ctx, out = B.from_array(np.full(q.shape, 7.25, np.float32)), B.from_array(np.full(q.shape[:2], 7.25, np.float32))
    rehip.attention_kv8_sinks_dev(B.from_array(full), ldq, *bt.args(), *cache.args(), max(max_rows, 1), max_len, heads,
                                  kv_heads, hd, scale, window, sinks, ctx, out if lse else None, work, nb, stream)
    hip.synchronize()
    return ctx.download(np.float32, q.size).reshape(q.shape), out.download(np.float32, rows * heads).reshape(rows, heads)


def near(got, want, tol):
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    np.testing.assert_array_equal(got == -np.inf, want == -np.inf)
    with np.errstate(invalid="ignore"):
        err = np.where(np.isfinite(want), np.abs(got - want), 0)
    assert np.all(err <= np.nan_to_num(tol, nan=np.inf)), (err.max(), np.unravel_index(err.argmax(), err.shape))


def check(cache, bt, q, scale, window, sinks, **k):
    ctx, lse = np.full(q.shape, 7.25), np.full(q.shape[:2], 7.25)
    tol, tol_lse = ref.attention(q, bt.plain(), (cache.k, cache.v, cache.ks, cache.vs), scale, window, sinks, ctx, lse)
    got, got_lse = attend_sinks(cache, bt, q, scale, window, sinks, **k)
    near(got, ctx, np.broadcast_to(tol[..., None], q.shape))
    near(got_lse, lse, tol_lse)
    return got, got_lse


# (rows of each request, tokens of each with them)
BATCHES = {
    "one token": ([1], [1]),
    "decode": ([1] * 10, [1, 2, 31, 32, 33, 64, 65, 127, 300, 900]),
    "drafts": ([5, 0, 3, 1, 5], [700, 7, 35, 1, 5]),
    "prompts": ([200, 3, 129, 64], [200, 67, 400, 128]),
    "one long": ([300], [1300]),
}
SHAPES = [(14, 2, 64, 32), (8, 1, 128, 64), (3, 3, 96, 96), (20, 1, 32, 64), (16, 2, 256, 32), (6, 2, 160, 128),
          (4, 1, 192, 256), (5, 5, 224, 64)]


@pytest.mark.parametrize("name", BATCHES)
@pytest.mark.parametrize("heads,kv_heads,hd,page", SHAPES)
@pytest.mark.parametrize("window,sinks", [(100, 4), (1, 1), (33, 70)])
def test_attention(name, heads, kv_heads, hd, page, window, sinks):
    rng = np.random.default_rng(heads + hd + page + window)
    bt, cache, q = make(rng, *BATCHES[name], page, heads, kv_heads, hd, gap=hd // 64 % 2)
    check(cache, bt, q, hd ** -0.5, window, sinks, ldq=heads * hd + 4)


@pytest.mark.parametrize("window,sinks", [(0, 0), (0, 9), (64, 0), (32, 32), (1, 1024), (5000, 3), (2, 31), (64, 64),
                                          (250, 33), (96, 96)])
@pytest.mark.parametrize("page", [32, 64, 256])
def test_windows_and_sinks(window, sinks, page):
    """Sinks that meet the window, that end in the middle of a step or a page, that are more than the request holds; none."""
    rng = np.random.default_rng(window + sinks + page)
    bt, cache, q = make(rng, [1, 40, 2, 1], [1290, 700, 33, 4], page, 6, 2, 64)
    got, _ = check(cache, bt, q, 0.125, window, sinks)
    if sinks == 0 or window == 0:        # the call without sinks gives the same bits
        np.testing.assert_array_equal(got, attend(cache, bt, q, 0.125, window))


@pytest.mark.parametrize("rows_of,len_of,window,sinks", [([1], [30000], 9000, 4), ([5, 1], [9000, 20000], 4096, 1000),
                                                         ([64], [12000], 6000, 40), ([1] * 70, [2000 + 37 * i for i in range(70)], 1500, 4)])
@pytest.mark.parametrize("heads,kv_heads,hd,page", [(8, 2, 128, 64), (4, 4, 32, 32)])
def test_long_requests(rows_of, len_of, window, sinks, heads, kv_heads, hd, page):
    """Windows cut into pieces of several workgroups, joined; more pages than are staged at a time."""
    rng = np.random.default_rng(len(rows_of) + window + hd)
    bt, cache, q = make(rng, rows_of, len_of, page, heads, kv_heads, hd)
    if len(rows_of) < 10:
        check(cache, bt, q, hd ** -0.5, window, sinks)
        return
    some = [0, 13, 69]                   # (the plain one takes long: a few of the requests)
    ctx, lse = attend_sinks(cache, bt, q, hd ** -0.5, window, sinks)
    want, want_lse = np.full(q.shape, 7.25), np.full(q.shape[:2], 7.25)
    start, count, kv_len, table, pg = bt.plain()
    tol, tol_lse = ref.attention(q, (start[some], count[some], kv_len[some], table[some], pg),
                                 (cache.k, cache.v, cache.ks, cache.vs), hd ** -0.5, window, sinks, want, want_lse)
    near(ctx[some], want[some], np.broadcast_to(tol[some][..., None], q[some].shape))
    near(lse[some], want_lse[some], tol_lse[some])


@pytest.mark.parametrize("requests,most", [(300, 60), (1000, 200)])
def test_many_requests(requests, most):
    """More requests than a workgroup looks at: pieces listed by a launch before, a wave for each of short ones."""
    rng = np.random.default_rng(requests)
    len_of = rng.integers(0, most + 1, requests)
    bt, cache, q = make(rng, np.minimum(len_of, 1), len_of, 32, 8, 4, 32)
    check(cache, bt, q, 0.2, 40, 5, max_len=most)


def test_wide_tiles_and_long_lists():
    """Tiles of 64 vectors, and decode steps of several rows over long windows in wide tiles."""
    rng = np.random.default_rng(5)
    bt, cache, q = make(rng, [700, 300], [900, 1100], 64, 32, 1, 64)
    some = np.r_[0:3, 350:353, 698:703, 990:1000]
    got, lse = attend_sinks(cache, bt, q, 0.125, 200, 6)
    want, wl = np.full(q.shape, 7.25), np.full(q.shape[:2], 7.25)
    start, count, kv_len, table, page = bt.plain()
    for r in some:                       # a request of its own for each row looked at
        b = 0 if r < 700 else 1
        p = kv_len[b] - count[b] + r - start[b]
        one = (np.array([r]), np.array([1]), np.array([p + 1]), table[b:b + 1], page)
        tol, tol_lse = ref.attention(q, one, (cache.k, cache.v, cache.ks, cache.vs), 0.125, 200, 6, want, wl)
        near(got[r], want[r], np.broadcast_to(tol[r][:, None], got[r].shape))
        near(lse[r], wl[r], tol_lse[r])


def test_rows_that_see_nothing():
    """Absent pages, tables of rubbish, windows behind the table, rows before position 0, rows past max_rows."""
    rng = np.random.default_rng(6)
    bt, cache, q = make(rng, [4, 3, 2, 6, 3], [90, 64, 2, 40, 300], 32, 4, 2, 32)
    bt.table[0] = -1
    bt.table[1, 0], bt.table[1, 1] = bt.n_pages, 1 << 30
    bt.table[4, 0] = -5                  # the sinks' page: the window alone is seen
    bt.len[3] = 4                        # two rows before position 0
    check(cache, bt, q, 0.2, 20, 4, max_len=300)
    bt.len[4] = bt.ld * 32 + 70          # the window is behind the table, the sinks are not
    bt.table[4, 0] = bt.table[4, 1]
    got, lse = check(cache, bt, q, 0.2, 20, 4, max_len=300)
    assert np.all(got[:4] == 0) and np.all(lse[:4] == -np.inf) and np.all(np.isfinite(lse[-3:]))
    got, lse = attend_sinks(cache, bt, q, 0.2, 20, 4, max_rows=2)
    assert np.all(got[2:4] == 7.25) and np.all(lse[2:4] == 7.25) and np.all(lse[0:2] == -np.inf)


def test_lse_may_be_left_out_and_huge_scores():
    rng = np.random.default_rng(7)
    bt, cache, q = make(rng, [3, 1, 90], [500, 77, 200], 64, 8, 2, 64)
    a, _ = attend_sinks(cache, bt, q, 0.125, 100, 4)
    b, lse = attend_sinks(cache, bt, q, 0.125, 100, 4, lse=False)
    np.testing.assert_array_equal(a, b)
    assert np.all(lse == 7.25)
    check(cache, bt, (q * 1e4).astype(np.float32), 3.0, 100, 4)
    check(cache, bt, q, -0.25, 100, 4)
    check(cache, bt, np.zeros_like(q), 0.125, 100, 4)
    q[2, 3, 5], q[10, 0, 0] = np.nan, np.inf
    got, lse = attend_sinks(cache, bt, q, 0.125, 100, 4)
    assert np.all(np.isnan(got[2, 3])) and np.isnan(lse[2, 3])
    rest = np.ones(q.shape[:2], bool)
    rest[2, 3] = rest[10, 0] = False
    assert np.all(np.isfinite(got[rest])) and np.all(np.isfinite(lse[rest]))


# ---- the weights of a step ---------------------------------------------------------------------
def weigh(cache, bt, q, lse, scale, window, sinks, masses, max_rows=None, max_len=None, stream=None, ldq=None):
    rows, heads, hd = q.shape
    ldq = ldq or heads * hd
    full = np.full((rows, ldq), np.nan, np.float32)
    full[:, :heads * hd] = q.reshape(rows, -1)
    buf = B.from_array(masses.astype(np.float32))
    rehip.kv8_mass_dev(B.from_array(full), ldq, B.from_array(lse), *bt.args(), cache.kb, cache.ksb,
                       int(max(bt.count.max(), 1)) if max_rows is None else max_rows,
                       int(bt.len.max()) if max_len is None else max_len, heads, cache.shape[1], hd, scale, window, sinks,
                       buf, stream)
    hip.synchronize()
    return buf.download(np.float32, masses.size).reshape(masses.shape)


def check_mass(cache, bt, q, scale, window, sinks, **k):
    rng = np.random.default_rng(99)
    _, lse = attend_sinks(cache, bt, q, scale, window, sinks)
    start = rng.random(cache.shape[:3]).astype(np.float32)
    want = start.astype(np.float64)
    tol = ref.mass(q, lse, bt.plain(), cache.k, cache.ks, scale, window, sinks, want)
    got = weigh(cache, bt, q, lse, scale, window, sinks, start, **k)
    err = np.abs(got - want)
    assert np.all(err <= tol), (err.max(), np.unravel_index((err - tol).argmax(), err.shape))
    assert np.array_equal(got, weigh(cache, bt, q, lse, scale, window, sinks, start, **k))      # one order of sums
    return got, start


@pytest.mark.parametrize("name", BATCHES)
@pytest.mark.parametrize("heads,kv_heads,hd,page", SHAPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 4)])
def test_mass(name, heads, kv_heads, hd, page, window, sinks):
    rng = np.random.default_rng(heads + hd + page + window + 1)
    bt, cache, q = make(rng, *BATCHES[name], page, heads, kv_heads, hd, gap=hd // 64 % 2)
    check_mass(cache, bt, q, hd ** -0.5, window, sinks, ldq=heads * hd + 4)


@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 1), (64, 300), (500, 33)])
@pytest.mark.parametrize("max_len", [1, 700, 5000])
def test_mass_planned_lengths(window, sinks, max_len):
    """max_len only decides how the work is cut; more vectors than a round of tiles, groups that divide no tile."""
    rng = np.random.default_rng(window + 7)
    bt, cache, q = make(rng, [3, 60, 1], [1290, 700, 40], 32, 15, 3, 64)
    check_mass(cache, bt, q, 0.125, window, sinks, max_len=max_len)


def test_mass_touches_its_tokens_alone():
    """Absent pages, tables of rubbish, idle requests, tokens behind the length and out of the window: left as they were;
    rows that are not finite add nothing."""
    rng = np.random.default_rng(8)
    bt, cache, q = make(rng, [4, 3, 0, 2, 2], [90, 64, 50, 41, 300], 32, 4, 2, 32)
    bt.table[0, 1] = -1
    bt.table[1, 0] = bt.n_pages
    q[0, 1, 3], q[1, 0, 0] = np.nan, -np.inf
    got, start = check_mass(cache, bt, q, 0.2, 33, 3)
    for b, lo, hi in ((3, 41, 64), (4, 3, 266), (2, 0, 64)):      # behind the length; between sinks and window; idle
        for j in range(lo, hi):
            np.testing.assert_array_equal(got[bt.table[b, j // 32], :, j % 32], start[bt.table[b, j // 32], :, j % 32])


def test_mass_sums_to_the_rows():
    """Every row and query head hands out a weight of one."""
    rng = np.random.default_rng(9)
    bt, cache, q = make(rng, [1, 77, 5], [1000, 400, 5], 64, 8, 2, 128)
    _, lse = attend_sinks(cache, bt, q, 0.1, 0, 0)
    got = weigh(cache, bt, q, lse, 0.1, 0, 0, np.zeros(cache.shape[:3]))
    # each weight to 2^-20 (lse below 16), each sum of below 800 to its roundings
    np.testing.assert_allclose(got.sum((0, 2), dtype=np.float64), 83 * 4, rtol=2.0 ** -18)
