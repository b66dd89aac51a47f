"""Calls at the edges of the batched serving entry points: pages that requests share, offsets past 32 bits, captured
graphs replayed between eager work, the largest sizes, wide tiles of odd queries."""
import ctypes as C

import numpy as np
import pytest

import rehip
import serving_ref as ref
from rehip import hip
from test_gpu_kv8 import Batch, Cache, append_both, attend, check_attention, i32, make
from test_gpu_serve_ops import EPS, Pool, check_logprobs, get, run_logprobs

pytestmark = pytest.mark.gpu
B = hip.DeviceBuffer


def put(address, a):
    """a copied to a device address"""
    a = np.ascontiguousarray(a)
    hip.check(hip.hip().hipMemcpy(C.c_void_p(address), a.ctypes.data, a.nbytes, hip.H2D))


# ---- pages ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows_of,len_of", [([1, 1, 1, 1], [200, 140, 129, 200]), ([30, 12, 1, 30], [200, 140, 129, 200])])
def test_requests_that_share_full_pages(rows_of, len_of):
    """Requests 0 .. 2 have their first 128 tokens in the same pages and append behind them; 3 is request 0's table once
    more and only reads."""
    rng = np.random.default_rng(30)
    bt, cache, q = make(rng, rows_of, len_of, 64, 8, 2, 64)
    bt.table[1, :2] = bt.table[2, :2] = bt.table[0, :2]
    k, v = (rng.standard_normal((bt.rows, 2, 64)).astype(np.float32) for _ in range(2))
    asked, bt.count = bt.count, bt.count.copy()
    bt.count[3] = 0
    append_both(cache, bt, k, v)
    cache.check()
    bt.count = asked
    bt.table[3] = bt.table[0]
    got = check_attention(cache, bt, q, 0.125)
    q[bt.start[3]:] = q[:asked[0]]
    got = attend(cache, bt, q, 0.125)
    np.testing.assert_array_equal(got[bt.start[3]:], got[:asked[0]])


def test_pages_past_32_bits():
    """A pool of 2 x 4.7 GB: pages from 2^32 bytes on give what the same pages of a small pool give."""
    rng = np.random.default_rng(31)
    page, hd, kv, heads, far = 256, 256, 8, 16, 9000
    size = kv * page * hd
    assert (far - 8) * size > 1 << 32
    rows_of, len_of = [300, 1, 40], [300, 1, 40]
    bt = Batch(rng, rows_of, len_of, page)
    k, v = (rng.standard_normal((bt.rows, kv * hd)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((bt.rows, heads * hd)).astype(np.float32)
    results = []
    for n_pages in (bt.n_pages, far):
        shift = n_pages - bt.n_pages
        table = np.where(bt.table >= 0, bt.table + shift, -1)
        cache = [B(n_pages * size), B(n_pages * size), B(n_pages * kv * 4), B(n_pages * kv * 4)]
        batch = (bt.rows, 3, i32(bt.start), i32(bt.count), i32(bt.len), i32(table), bt.ld, page, n_pages, *cache)
        nb = rehip.attention_kv8_work_bytes(bt.rows, 3, 300, 300, heads, kv, hd)
        work, ctx = B(max(nb, 16)), B(bt.rows * heads * hd * 4)
        rehip.kv8_append_dev(B.from_array(k), kv * hd, B.from_array(v), kv * hd, *batch, kv, hd)
        rehip.attention_kv8_dev(B.from_array(q), heads * hd, *batch, 300, 300, heads, kv, hd, 1 / 16, 0, ctx, work, nb)
        one = [i32([0]), i32([1]), i32([300]), i32(table[:1])]
        more = B(heads * hd * 4)
        nb = rehip.attention_kv8_work_bytes(1, 1, 1, 300, heads, kv, hd)
        rehip.attention_kv8_dev(B.from_array(q[299:300]), heads * hd, 1, 1, *one, bt.ld, page, n_pages, *cache, 1, 300,
                                heads, kv, hd, 1 / 16, 0, more, B(max(nb, 16)), nb)
        results.append((get(ctx, q.size), get(more, heads * hd)))
        for b in cache:
            b.free()
    for a, b in zip(*results):
        np.testing.assert_array_equal(a, b)
    assert np.all(np.isfinite(results[0][0]))


def test_append_of_odd_values_in_large_pages():
    """Pages of more units than threads hold: infinities, NaN and a growing scale there too."""
    rng = np.random.default_rng(32)
    page, hd, h = 256, 160, 2
    bt = Batch(rng, [100, 30, 5], [100, 290, 200], page)
    cache = Cache(rng, bt.n_pages, h, page, hd)
    cache.ks *= np.float32(1e-2)
    cache.upload()
    k, v = (rng.standard_normal((bt.rows, h, hd)).astype(np.float32) for _ in range(2))
    k[3, 0, 7], v[99, 1, 159], k[110, 1, 0], v[131, 0, 3] = np.inf, -np.inf, np.nan, np.inf
    v[0:100, 0] *= np.float32(1e-37)
    append_both(cache, bt, k, v)
    cache.check()


@pytest.mark.parametrize("page,hd,kv_heads", [(32, 64, 5), (64, 128, 9), (256, 160, 3), (96, 256, 4), (64, 32, 1)])
def test_append_of_a_decode_step_with_a_prompt_in_it(page, hd, kv_heads):
    """No more rows than requests, but not one each: some idle, some with a few, one with more than a page; then tokens one by
    one, with scales that grow and stay, infinities and NaN among them."""
    rng = np.random.default_rng(page + hd)
    n = 450
    rows_of = np.zeros(n, int)
    rows_of[[3, 7, 70, 200, 449]] = 1, 9, page + 40, 3, 1
    rows_of[100:180] = 1
    rows_of[300:306] = 2
    len_of = rows_of + rng.integers(0, 2 * page, n)
    bt = Batch(rng, rows_of, len_of, page, spare=2)
    assert bt.rows <= n
    cache = Cache(rng, bt.n_pages, kv_heads, page, hd)
    for turn in range(4):
        k, v = ((rng.standard_normal((bt.rows, kv_heads, hd)) * np.exp(2 * rng.standard_normal((bt.rows, kv_heads, 1))))
                .astype(np.float32) for _ in range(2))
        k[rng.integers(0, bt.rows, 5), 0, 3] = np.inf
        v[rng.integers(0, bt.rows, 5), kv_heads - 1, hd - 1] = np.nan
        append_both(cache, bt, k, v)
        cache.check()
        bt.len = np.minimum(bt.len + 1, bt.ld * page).astype(np.int32)
        bt.count = np.minimum(bt.count, 1).astype(np.int32)


@pytest.mark.parametrize("n", [64, 65, 200, 4096, 4097, 5000])
def test_batches_of_many_requests(n):
    """Requests on both sides of every step of the search for a request, most idle, unused rows among them."""
    rng = np.random.default_rng(n)
    rows_of = (rng.random(n) < 0.3) * rng.integers(1, 4, n)
    rows_of[n - 1] = 2
    bt = Batch(rng, rows_of, rows_of + rng.integers(0, 40, n), 32)
    cache = Cache(rng, bt.n_pages, 1, 32, 32)
    k, v = (rng.standard_normal((bt.rows, 1, 32)).astype(np.float32) for _ in range(2))
    append_both(cache, bt, k, v)
    cache.check()
    q = rng.standard_normal((bt.rows, 20, 32)).astype(np.float32)   # (20 heads a row: tiles of one row or two)
    cache.ks *= np.float32(0.02)
    cache.upload()
    check_attention(cache, bt, q, 0.2)


@pytest.mark.parametrize("n", [200, 300, 1100, 4100])
@pytest.mark.parametrize("page,max_len", [(64, 4000), (64, 60000), (64, 2000), (32, 100)])
def test_many_requests_and_a_few_long_ones(n, page, max_len):
    """Pieces of a few long requests among many short, idle and empty ones; few splits, many and none (planned for)."""
    rng = np.random.default_rng(n)
    len_of = rng.integers(1, 40, n)
    len_of[[5, n // 2, n - 1]] = 4000, 2111, 1500
    rows_of = (rng.random(n) < 0.6).astype(int)
    rows_of[[5, n // 2, n - 1]] = 1
    rows_of[7], len_of[7] = 1, 0                            # (a row before the first token)
    bt, cache, q = make(rng, rows_of, len_of, page, 6, 2, 64)
    check_attention(cache, bt, q, 0.125, max_len=max_len)
    check_attention(cache, bt, q, 0.125, 1000, max_len=max_len)
    bt.count[:] = 0
    bt.count[n // 2] = 1
    check_attention(cache, bt, q, 0.125, max_len=max_len)


# ---- offsets past 32 bits of rows ------------------------------------------------------------------
def test_row_strides_past_32_bits():
    """Three rows 2^30 floats apart (the third begins at byte 2^33): log probabilities, rotary positions, attention."""
    rng = np.random.default_rng(33)
    ld, vocab = 1 << 30, 5000
    big = B(4 * (2 * ld + 8192))
    x = rng.standard_normal((3, vocab)).astype(np.float32)
    at = lambda r: big.ptr + 4 * ld * r  # noqa: E731
    for r in range(3):
        put(at(r), x[r])
    nb = rehip.logprobs_work_bytes(3, vocab, 9)
    work, lp, en, ids, top = B(max(nb, 16)), B(12), B(12), B(108), B(108)
    rehip.logprobs_dev(big, ld, 3, vocab, i32([1, 2, 3]), 9, lp, en, ids, top, work, nb)
    want = run_logprobs(x, np.array([1, 2, 3]), 9)
    for got, w in zip((get(lp, 3), get(en, 3), get(ids, 27, np.int32), get(top, 27)), want):
        np.testing.assert_array_equal(got, w.reshape(-1))

    freqs, m = rehip.rope_freqs(1e4, 64)
    small, pos = B.from_array(x[:, :512]), i32([5, 9, 70000])
    for buf, stride in ((small, 512), (big, ld)):
        rehip.rope_rows_dev(buf, stride, 3, 8, 64, 64, rehip.ROPE_HALF, B.from_array(freqs), m, pos, buf, stride)
    turned = get(small, 3 * 512).reshape(3, 512)
    back = np.empty((3, 512), np.float32)
    for r in range(3):
        hip.check(hip.hip().hipMemcpy(back[r].ctypes.data, C.c_void_p(at(r)), 2048, hip.D2H))
    np.testing.assert_array_equal(back, turned)

    bt, cache, q = make(rng, [1, 2], [200, 90], 32, 8, 2, 64)
    for r in range(3):
        put(at(r), q[r])
    want = attend(cache, bt, q, 0.125)
    nb = rehip.attention_kv8_work_bytes(3, 2, 2, 200, 8, 2, 64)
    ctx = B(q.nbytes)
    rehip.attention_kv8_dev(big, ld, *bt.args(), *cache.args(), 2, 200, 8, 2, 64, 0.125, 0, ctx, B(max(nb, 16)), nb)
    np.testing.assert_array_equal(get(ctx, q.size).reshape(q.shape), want)
    big.free()


# ---- graphs --------------------------------------------------------------------------------------
def test_two_graphs_with_workspaces_of_their_own():
    """Attention over a long context and log probabilities, each captured on a stream of its own, replayed in turn and
    at once, with eager calls between: every replay gives the eager result."""
    rng = np.random.default_rng(34)
    bt, cache, q = make(rng, [1, 1], [9000, 70], 64, 8, 1, 64)
    want_ctx = attend(cache, bt, q, 0.125)
    x = rng.standard_normal((5, 40000)).astype(np.float32)
    want_lp = run_logprobs(x, np.arange(5), 7)
    nb = rehip.attention_kv8_work_bytes(2, 2, 1, 9000, 8, 1, 64)
    assert nb > 0
    qb, ctx, awork, abatch = B.from_array(q), B(q.nbytes), B(nb), (*bt.args(), *cache.args())
    lb = rehip.logprobs_work_bytes(5, 40000, 7)
    assert lb > 0
    xb, tb, lwork = B.from_array(x), i32(np.arange(5)), B(lb)
    lp, en, ids, top = B(20), B(20), B(140), B(140)
    s, u = hip.Stream(), hip.Stream()
    g = hip.Graph(s, lambda: rehip.attention_kv8_dev(qb, 512, *abatch, 1, 9000, 8, 1, 64, 0.125, 0, ctx, awork, nb, s))
    h = hip.Graph(u, lambda: rehip.logprobs_dev(xb, 40000, 5, 40000, tb, 7, lp, en, ids, top, lwork, lb, u))

    def clean():
        ctx.upload(np.full(q.shape, 3.0, np.float32))
        for b in (awork, lwork):
            b.upload(np.full(b.nbytes // 4, np.nan, np.float32))
        for b in (lp, en, ids, top):
            b.upload(np.full(b.nbytes // 4, 3.0, np.float32))
        hip.synchronize()

    for turn in range(6):
        clean()
        g.launch()
        if turn % 2:
            s.synchronize()
        h.launch()
        if turn % 3 == 0:
            np.testing.assert_array_equal(attend(cache, bt, q, 0.125), want_ctx)
        hip.synchronize()
        np.testing.assert_array_equal(ctx.download(np.float32, q.size).reshape(q.shape), want_ctx)
        for got, w in zip((get(lp, 5), get(en, 5), get(ids, 35, np.int32), get(top, 35)), want_lp):
            np.testing.assert_array_equal(got, w.reshape(-1))
    g.destroy()
    h.destroy()


# ---- sizes ---------------------------------------------------------------------------------------
def test_logprobs_of_the_largest_vocabulary():
    """2^24 logits: a lane adds 1024 terms and the joins some tens, each rounded once."""
    rng = np.random.default_rng(35)
    vocab = 1 << 24
    x = rng.standard_normal((1, vocab)).astype(np.float32)
    x[0, [5, vocab - 1]] = 9.0
    got, want = run_logprobs(x, np.array([vocab - 1]), 64), ref.logprobs(x, np.array([vocab - 1]), 64)
    np.testing.assert_array_equal(got[2], want[2])
    assert got[2][0, :2].tolist() == [5, vocab - 1]
    tol = (1024 + 100) * EPS + 4 * EPS * 20
    assert abs(got[0][0] - want[0][0]) <= tol and np.all(np.abs(got[3] - want[3]) <= tol)
    assert abs(got[1][0] - want[1][0]) <= tol * (1 + np.log(vocab))


def test_nothing_to_do():
    """Batches without rows or requests, requests without rows, a planned length of 0: outputs are left or zero."""
    rng = np.random.default_rng(36)
    bt, cache, q = make(rng, [3, 2], [50, 2], 32, 4, 2, 64)
    bt.count[:] = 0
    assert np.all(attend(cache, bt, q, 0.125, max_len=0) == 7.25)
    before = cache.k.copy()
    rehip.kv8_append_dev(B.from_array(q[:, :2]), 128, B.from_array(q[:, :2]), 128, *bt.args(), *cache.args(), 2, 64)
    args = bt.args()
    for rows, requests in ((0, 2), (5, 0)):
        rehip.kv8_append_dev(B.from_array(q[:, :2]), 128, B.from_array(q[:, :2]), 128, rows, requests, *args[2:],
                             *cache.args(), 2, 64)
    hip.synchronize()
    got = ref.unpack(cache.kb.download(np.int8, before.size), *cache.shape, 0)
    np.testing.assert_array_equal(got, before)
    bt.count[:] = [3, 2]
    check_attention(cache, bt, q, 0.125, max_len=0)


def test_plan_of_more_pages_than_the_pool_has():
    """Ended requests whose tables claim pages while the stack is full: the stack stays in its array."""
    p = Pool(3, 32, 4, 6, np.random.default_rng(37))
    p.len[:] = [100, 64, 128]                               # (of pages that were never taken)
    p.table[:] = np.arange(12).reshape(3, 4)
    p.dev.update(len=i32(p.len), table=i32(p.table))
    assert p.step([-1, -1, 5], 10)["n_free"] == 6           # (request 2 has no room in its table)
    assert p.step([33, 0, -1], 40)["n_free"] == 4


def test_rope_at_the_last_positions():
    """Positions up to 2^31 - 1. Beside the 12 roundings of test_rope_rows: the turns, up to 3.4e8, are off by three
    roundings of 2^-53 (3 * 2^-53 * 3.4e8 * 2 pi: 12 EPS), the plain angle by one (4 EPS)."""
    rng = np.random.default_rng(38)
    pos = np.array([2**31 - 1, 2**31 - 2, 1 << 30, 123456789], np.int32)
    x = rng.standard_normal((4, 2, 64)).astype(np.float32)
    freqs, m = rehip.rope_freqs(1e4, 64)
    for interleaved in (False, True):
        want = ref.rope(x, pos, freqs, m, 64, interleaved)
        out = B(x.nbytes)
        rehip.rope_rows_dev(B.from_array(x), 128, 4, 2, 64, 64, rehip.ROPE_INTERLEAVED if interleaved else rehip.ROPE_HALF,
                            B.from_array(freqs), m, i32(pos), out, 128)
        np.testing.assert_allclose(get(out, x.size).reshape(x.shape), want, rtol=0,
                                   atol=(12 + 16) * EPS * 3 * np.abs(x).max())


# ---- wide tiles ----------------------------------------------------------------------------------
@pytest.mark.parametrize("heads,kv_heads,hd", [(14, 2, 64), (5, 1, 32), (40, 2, 96), (16, 2, 256), (3, 3, 160)])
def test_waves_alone(heads, kv_heads, hd):
    """Many short requests, a wave each: odd queries, holes, windows, groups of more heads than a tile has vectors."""
    rng = np.random.default_rng(hd)
    n = 270
    len_of = rng.integers(0, 70, n)
    len_of[::50] = rng.integers(300, 600, 6)               # (the others' length is planned for)
    bt, cache, q = make(rng, np.ones(n, int), len_of, 32, heads, kv_heads, hd, gap=1)
    live = np.flatnonzero(len_of > 0)
    q[bt.start[live[0]], 0, 3], q[bt.start[live[1]], heads - 1, 0], q[bt.start[live[2]]] = np.nan, np.inf, 0
    bt.table[live[3], 0], bt.table[live[4]] = -1, bt.n_pages
    check_attention(cache, bt, q, hd ** -0.5, max_len=60)
    check_attention(cache, bt, q, -hd ** -0.5, 40, max_len=64)
    check_attention(cache, bt, q, hd ** -0.5, max_len=600)


def test_odd_queries_in_wide_tiles():
    """Tiles of 64 vectors with queries of NaN, infinities, zeros and huge scores: each spoils its own row and head only,
    and scores past 2^20 keep their neighbours' precision."""
    rng = np.random.default_rng(39)
    bt, cache, q = make(rng, [200, 63], [230, 64], 32, 256, 64, 32)
    q[0, 1, 3], q[1, 5, 0], q[2, 7] = np.nan, np.inf, 0
    q[3] *= np.float32(1e-30)
    q[40:50] *= np.float32(1e20)
    cache.vs[bt.table[0, 0]] = 0
    cache.ks[bt.table[0, 1], 0] = 0
    cache.vs[bt.table[1, 1]] *= np.float32(1e-12)
    cache.upload()
    want = np.full(q.shape, 7.25)
    tol = ref.attention(q, *bt.plain(), cache.k, cache.v, cache.ks, cache.vs, 0.125, 0, want)
    got = attend(cache, bt, q, 0.125)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    fine = ~np.isnan(want)
    huge = np.zeros(q.shape, bool)
    huge[40:50] = True                                      # a softmax of one key, unless two scores are close
    rest = fine & ~huge
    assert np.all(np.abs(got - want)[rest] <= np.broadcast_to(tol[..., None], want.shape)[rest])
    # (a huge row's output is still a mean of values, up to 128 scales each, off by its few hundred roundings)
    assert np.all(np.abs(got[huge]) <= 128 * cache.vs.max() * (1 + 2.0 ** -14))


def test_logprobs_rows_between_the_forms():
    """Row counts on both sides of every change of form agree with the plain form."""
    rng = np.random.default_rng(40)
    for rows, vocab in ((1535, 1025), (1536, 1025), (3, 1024), (3, 1025), (384, 9000), (385, 9000), (768, 4097)):
        x = (2 * rng.standard_normal((rows, vocab))).astype(np.float32)
        check_logprobs(x, rng.integers(0, vocab, rows), 3)
