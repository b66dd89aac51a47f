"""The paged int8 K/V cache: append (bit for bit) and attention, against the plain restatements of
serving_ref.py, at ragged batches, part-filled pages, absent pages, empty rows and values that must not leak."""
import numpy as np
import pytest

import rehip
import serving_ref as ref
from rehip import hip

pytestmark = pytest.mark.gpu
B = hip.DeviceBuffer


def i32(a):
    return B.from_array(np.ascontiguousarray(a, np.int32))


class Cache:
    """Pages on the device and the same pages in rows; everything starts as rubbish."""

    def __init__(self, rng, n_pages, kv_heads, page, hd):
        self.shape = (n_pages, kv_heads, page, hd)
        self.k, self.v = (rng.integers(-128, 128, self.shape).astype(np.int8) for _ in range(2))
        self.ks, self.vs = (np.exp(2 * rng.standard_normal((n_pages, kv_heads))).astype(np.float32) for _ in range(2))
        self.upload()

    def upload(self):
        self.kb, self.vb = (B.from_array(ref.pack(c, v)) for c, v in ((self.k, 0), (self.v, 1)))
        self.ksb, self.vsb = B.from_array(self.ks), B.from_array(self.vs)

    def args(self):
        return self.kb, self.vb, self.ksb, self.vsb

    def check(self):
        hip.synchronize()
        n, h, page, hd = self.shape
        size = n * h * page * hd
        np.testing.assert_array_equal(ref.unpack(self.kb.download(np.int8, size), n, h, page, hd, 0), self.k)
        np.testing.assert_array_equal(ref.unpack(self.vb.download(np.int8, size), n, h, page, hd, 1), self.v)
        np.testing.assert_array_equal(self.ksb.download(np.float32, n * h), self.ks.reshape(-1))
        np.testing.assert_array_equal(self.vsb.download(np.float32, n * h), self.vs.reshape(-1))


class Batch:
    """rows_of / len_of: new rows and tokens of each request; pages shuffled, `gap` unused rows between requests."""

    def __init__(self, rng, rows_of, len_of, page, gap=0, spare=2, ld_extra=1):
        self.count, self.len = np.asarray(rows_of, np.int32), np.asarray(len_of, np.int32)
        n = len(rows_of)
        need = -(-np.maximum(self.len, 0) // page)
        self.n_pages, self.ld, self.page = int(need.sum()) + spare, int(need.max()) + ld_extra, page
        order = rng.permutation(self.n_pages)
        self.table = np.full((n, self.ld), -1, np.int32)
        at = 0
        for b in range(n):
            self.table[b, :need[b]] = order[at:at + need[b]]
            at += need[b]
        self.start = (np.concatenate([[0], np.cumsum(np.maximum(self.count, 0) + gap)])[:-1]).astype(np.int32)
        self.rows = int(self.start[-1] + max(self.count[-1], 0) + gap)

    def args(self):
        return (self.rows, len(self.count), i32(self.start), i32(self.count), i32(self.len), i32(self.table), self.ld,
                self.page, self.n_pages)

    def plain(self):
        return self.start, self.count, self.len, self.table, self.page


def append_both(cache, bt, k, v, ldk=None, ldv=None):
    """The library's append on the device pages, the plain one on the others; strided inputs."""
    rows, h, hd = k.shape
    def strided(x, ld):
        full = np.full((rows, ld), 1e30, np.float32)
        full[:, :h * hd] = x.reshape(rows, -1)
        return B.from_array(full)
    ldk, ldv = ldk or h * hd, ldv or h * hd
    rehip.kv8_append_dev(strided(k, ldk), ldk, strided(v, ldv), ldv, *bt.args(), *cache.args(), h, hd)
    ref.append(k, *bt.plain(), cache.k, cache.ks)
    ref.append(v, *bt.plain(), cache.v, cache.vs)


# (rows of each request, tokens of each with them)
BATCHES = {
    "one token": ([1], [1]),
    "decode": ([1] * 9, [1, 2, 31, 32, 33, 64, 65, 127, 300]),
    "idle and new": ([0, 5, 0, 1, 40, 0], [7, 5, 0, 33, 41, 90]),
    "prompts": ([200, 3, 129, 64], [200, 67, 400, 128]),
    "one long": ([517], [1300]),
}


@pytest.mark.parametrize("name", BATCHES)
@pytest.mark.parametrize("page,hd,kv_heads", [(32, 64, 2), (64, 128, 3), (64, 32, 1), (96, 96, 2), (128, 160, 1),
                                              (256, 256, 2)])
def test_append(name, page, hd, kv_heads):
    rng = np.random.default_rng(page + hd)
    rows_of, len_of = BATCHES[name]
    bt = Batch(rng, rows_of, len_of, page, gap=hd // 64 % 2)
    cache = Cache(rng, bt.n_pages, kv_heads, page, hd)
    k, v = ((rng.standard_normal((bt.rows, kv_heads, hd)) * np.exp(2 * rng.standard_normal((bt.rows, kv_heads, 1))))
            .astype(np.float32) for _ in range(2))
    append_both(cache, bt, k, v, ldk=kv_heads * hd + 4, ldv=3 * kv_heads * hd)
    cache.check()


def test_append_token_by_token():
    """A page filled one token at a time, the scale growing now and then; then the same tokens' earlier end again
    (kv_len set back), and a second page."""
    rng = np.random.default_rng(8)
    page, hd, h = 64, 64, 2
    bt = Batch(rng, [1], [70], page)
    cache = Cache(rng, bt.n_pages, h, page, hd)
    for t in list(range(1, 71)) + [20, 21, 22]:
        bt.len[0] = t
        k, v = ((rng.standard_normal((1, h, hd)) * 1.05 ** (t % 30)).astype(np.float32) for _ in range(2))
        append_both(cache, bt, k, v)
    cache.check()


def test_append_of_odd_values():
    """Zeros, values too small for a scale, the largest floats, infinities and NaN: stored as documented, the page's
    other tokens as without them."""
    rng = np.random.default_rng(9)
    page, hd, h = 32, 64, 3
    bt = Batch(rng, [10, 10, 10, 10, 10, 4], [12, 10, 42, 33, 10, 14], page)
    cache = Cache(rng, bt.n_pages, h, page, hd)
    k, v = (rng.standard_normal((bt.rows, h, hd)).astype(np.float32) for _ in range(2))
    k[0:10] = 0
    k[10:20] *= np.float32(1e-39)
    v[0:10] *= np.float32(3e-37)
    k[20, 1, 5], k[22, 0, 63], v[23, 2, 0] = np.inf, -np.inf, np.nan
    v[30:40] = np.nan
    k[30:40] = np.where(rng.random((10, h, hd)) < 0.5, np.inf, -np.inf)
    k[40, 0, 0], v[41, 1, 1] = np.finfo(np.float32).max, -np.finfo(np.float32).max
    append_both(cache, bt, k, v)
    cache.check()
    assert np.all(np.isfinite(cache.ks)) and np.all(np.isfinite(cache.vs))


def test_append_skips_what_has_no_place():
    """Absent pages, tables of rubbish, lengths that do not fit: skipped, nothing else touched."""
    rng = np.random.default_rng(10)
    page, hd, h = 32, 32, 2
    bt = Batch(rng, [40, 3, 50, 7, 2], [100, 3, 60, 7, 5], page, gap=2)
    bt.table[0, 2] = -1
    bt.table[1, 0] = bt.n_pages
    bt.table[3, 0] = 1 << 30
    bt.len[2], bt.len[4] = 49, bt.ld * page + 1
    cache = Cache(rng, bt.n_pages, h, page, hd)
    k, v = (rng.standard_normal((bt.rows, h, hd)).astype(np.float32) for _ in range(2))
    append_both(cache, bt, k, v)
    cache.check()


# ---- attention ---------------------------------------------------------------------------------
def attend(cache, bt, q, scale, window=0, max_rows=None, max_len=None, stream=None, ldq=None, work=None):
    rows, heads, hd = q.shape
    kv_heads = cache.shape[1]
    ldq = ldq or heads * hd
    full = np.full((rows, ldq), np.nan, np.float32)
    full[:, :heads * hd] = q.reshape(rows, -1)
    max_rows = int(bt.count.max()) if max_rows is None else max_rows
    max_len = int(bt.len.max()) if max_len is None else max_len
    nb = rehip.attention_kv8_work_bytes(rows, len(bt.count), max(max_rows, 1), max_len, heads, kv_heads, hd)
    work = work or B.from_array(np.full(max(nb // 4, 4), np.nan, np.float32))
    ctx = B.from_array(np.full(q.shape, 7.25, np.float32))
    rehip.attention_kv8_dev(B.from_array(full), ldq, *bt.args(), *cache.args(), max(max_rows, 1), max_len, heads,
                            kv_heads, hd, scale, window, ctx, work, nb, stream)
    hip.synchronize()
    return ctx.download(np.float32, q.size).reshape(q.shape)


def check_attention(cache, bt, q, scale, window=0, **k):
    want = np.full(q.shape, 7.25)
    tol = ref.attention(q, *bt.plain(), cache.k, cache.v, cache.ks, cache.vs, scale, window, want)
    got = attend(cache, bt, q, scale, window, **k)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    err = np.where(np.isnan(want), 0, np.abs(got - want))
    assert np.all(err <= np.nan_to_num(tol, nan=np.inf)[..., None]), (err.max(), np.unravel_index(err.argmax(), err.shape))
    return got


def make(rng, rows_of, len_of, page, heads, kv_heads, hd, gap=0):
    bt = Batch(rng, rows_of, len_of, page, gap)
    cache = Cache(rng, bt.n_pages, kv_heads, page, hd)
    cache.ks, cache.vs = ((0.03 * np.exp(0.5 * rng.standard_normal(s.shape))).astype(np.float32)
                          for s in (cache.ks, cache.vs))
    cache.upload()
    return bt, cache, (1.5 * rng.standard_normal((bt.rows, heads, hd))).astype(np.float32)


SHAPES = [(14, 2, 64, 32), (8, 1, 128, 64), (3, 3, 96, 96), (20, 1, 32, 64), (16, 2, 256, 32), (6, 2, 160, 128),
          (4, 1, 192, 256), (5, 5, 224, 64), (34, 1, 64, 64)]


@pytest.mark.parametrize("heads,kv_heads,hd,page", SHAPES)
@pytest.mark.parametrize("name", BATCHES)
def test_attention(heads, kv_heads, hd, page, name):
    rng = np.random.default_rng(heads * hd + page)
    rows_of, len_of = BATCHES[name]
    if name in ("prompts", "one long"):                     # (the plain form is a loop)
        rows_of, len_of = ([33, 3, 20, 64], [33, 67, 400, 128]) if name == "prompts" else ([41], [1300])
    bt, cache, q = make(rng, rows_of, len_of, page, heads, kv_heads, hd, gap=1)
    check_attention(cache, bt, q, hd ** -0.5, ldq=heads * hd + 8)


@pytest.mark.parametrize("heads,kv_heads,hd,page,rows_of,len_of", [
    (256, 64, 32, 32, [200, 1, 63], [230, 40, 64]),        # 64 vectors a tile: 16 rows of 4 heads
    (128, 128, 64, 64, [300, 260], [300, 500]),            # .. 64 rows of one
    (392, 56, 128, 64, [100, 70], [130, 70]),              # .. 9 rows of 7, one place unused
    (256, 64, 160, 32, [100, 33, 17], [100, 34, 90]),      # 32 vectors: 8 rows of 4
    (400, 20, 96, 96, [150, 1], [151, 1])])                 # 3 rows of 20 heads: 60 of 64
@pytest.mark.parametrize("window", [0, 37])
def test_attention_of_many_tiles(heads, kv_heads, hd, page, rows_of, len_of, window):
    """Enough tiles for wide ones (32 or 64 query vectors)."""
    rng = np.random.default_rng(hd)
    bt, cache, q = make(rng, rows_of, len_of, page, heads, kv_heads, hd, gap=2)
    check_attention(cache, bt, q, hd ** -0.5, window)


@pytest.mark.parametrize("heads,kv_heads,hd,rows_of", [(8, 1, 128, [4, 3, 4, 0, 1]), (14, 2, 64, [9, 5, 1, 9, 8]),
                                                       (20, 1, 256, [1, 1, 1, 0, 1]), (34, 2, 32, [3, 3, 1, 2, 3])])
def test_attention_of_wide_single_tiles(heads, kv_heads, hd, rows_of):
    """All rows of a request in one tile of 32 or 64 vectors, cut into pieces (max_len says that there is work for many)."""
    rng = np.random.default_rng(heads)
    len_of = [900, 4, 77, 0, 1500]
    bt, cache, q = make(rng, rows_of, len_of, 64, heads, kv_heads, hd, gap=1)
    for max_len in (1500, 1 << 20):
        check_attention(cache, bt, q, hd ** -0.5, max_len=max_len)
    check_attention(cache, bt, q, hd ** -0.5, 200, max_len=1 << 20)


def test_attention_of_many_requests():
    """More requests than a workgroup has threads, some without rows, in one launch; each wave of lengths 1 .. 60."""
    rng = np.random.default_rng(21)
    n = 700
    rows_of = rng.integers(0, 2, n)
    len_of = np.maximum(rng.integers(1, 61, n), rows_of)
    bt, cache, q = make(rng, rows_of, len_of, 32, 2, 1, 32)
    check_attention(cache, bt, q, 0.3)
    bt, cache, q = make(rng, rows_of * rng.integers(1, 4, n), len_of + 3, 32, 2, 1, 32, gap=1)
    check_attention(cache, bt, q, 0.3)


def test_append_of_many_requests():
    rng = np.random.default_rng(22)
    n = 700
    rows_of = rng.integers(0, 3, n)
    bt = Batch(rng, rows_of, rows_of + rng.integers(0, 60, n), 32, gap=1)
    cache = Cache(rng, bt.n_pages, 1, 32, 32)
    k, v = (rng.standard_normal((bt.rows, 1, 32)).astype(np.float32) for _ in range(2))
    append_both(cache, bt, k, v)
    cache.check()


def test_starts_that_do_not_ascend_stay_in_bounds():
    """Rows of such a batch may be skipped; nothing outside the arrays is touched and other pages keep their codes."""
    rng = np.random.default_rng(23)
    bt, cache, q = make(rng, [3, 2, 4, 1], [50, 2, 64, 33], 32, 4, 2, 64)
    bt.start[:] = [9, -5, 1 << 30, 3]
    k = rng.standard_normal((bt.rows, 2, 64)).astype(np.float32)
    other = np.setdiff1d(np.arange(bt.n_pages), bt.table[bt.table >= 0])
    kc, vc = cache.k.copy(), cache.v.copy()
    rehip.kv8_append_dev(B.from_array(k), 128, B.from_array(k), 128, *bt.args(), *cache.args(), 2, 64)
    hip.synchronize()
    for buf, was, is_v in ((cache.kb, kc, 0), (cache.vb, vc, 1)):
        got = ref.unpack(buf.download(np.int8, was.size), *cache.shape, is_v)
        np.testing.assert_array_equal(got[other], was[other])
    attend(cache, bt, q, 0.1)


@pytest.mark.parametrize("window", [1, 2, 31, 64, 100, 1000])
@pytest.mark.parametrize("heads,kv_heads,hd,page", [(8, 2, 64, 32), (14, 2, 128, 64)])
def test_attention_window(heads, kv_heads, hd, page, window):
    rng = np.random.default_rng(window)
    bt, cache, q = make(rng, [1, 40, 1, 7, 70], [700, 40, 1, 300, 170], page, heads, kv_heads, hd)
    check_attention(cache, bt, q, 0.11, window)


@pytest.mark.parametrize("max_len", [1, 100, 5000, 1 << 17])
def test_attention_plans_for_other_lengths(max_len):
    """max_len plans the split of the keys and nothing else; rows past max_rows are left."""
    rng = np.random.default_rng(4)
    bt, cache, q = make(rng, [1, 1, 1, 1], [2500, 1, 640, 129], 64, 8, 2, 64)
    check_attention(cache, bt, q, 0.125, max_len=max_len)
    bt, cache, q = make(rng, [9, 1, 30], [2500, 1, 640], 64, 8, 2, 64)
    want = check_attention(cache, bt, q, 0.125, max_len=max_len)
    got = attend(cache, bt, q, 0.125, max_rows=4, max_len=max_len)
    for b in range(3):
        s, n = bt.start[b], bt.count[b]
        # (fewer rows per request may split the keys elsewhere: another order of the sums)
        np.testing.assert_allclose(got[s:s + min(n, 4)], want[s:s + min(n, 4)], rtol=0, atol=2e-4 * np.abs(want).max())
        assert np.all(got[s + 4:s + n] == 7.25)


def test_attention_long():
    """Past 32768 tokens, where the f32 cache ends; all heads of a group, one row."""
    rng = np.random.default_rng(6)
    bt, cache, q = make(rng, [1, 2], [70001, 40000], 128, 4, 1, 32)
    check_attention(cache, bt, q, 0.2)


def test_attention_empty_rows_and_absent_pages():
    """Rows before position 0, requests without tokens or pages: zeros; holes in a table are not seen."""
    rng = np.random.default_rng(7)
    bt, cache, q = make(rng, [5, 3, 1, 2, 70], [200, 3, 40, 64, 300], 32, 6, 2, 64)
    bt.len[1] = 1                                           # two rows stand before the first token
    bt.table[0, 1], bt.table[0, 3] = -1, bt.n_pages
    bt.table[2] = -1
    bt.table[3, 0] = -1
    bt.table[4, 0:5] = 1 << 28                              # the first of 70 rows see only holes
    got = check_attention(cache, bt, q, 0.1)
    assert not got[bt.start[1]:bt.start[1] + 2].any() and not got[bt.start[2]].any()
    bt.len[:] = 0
    assert not attend(cache, bt, q, 0.1, max_len=300).any()


@pytest.mark.parametrize("rows_of,len_of", [([1, 1], [45, 200]), ([30, 40], [45, 200])])
def test_attention_hidden_values_do_not_leak(rows_of, len_of):
    """Codes behind a request's end and pages of others may hold anything; scales of pages that are not in the
    table may be NaN."""
    rng = np.random.default_rng(11)
    bt, cache, q = make(rng, rows_of, len_of, 64, 8, 2, 64)
    want = attend(cache, bt, q, 0.125)
    used = bt.table[bt.table >= 0]
    other = np.setdiff1d(np.arange(bt.n_pages), used)
    cache.ks[other], cache.vs[other] = np.nan, np.inf
    for b in range(2):
        last, at = bt.table[b, (len_of[b] - 1) // 64], len_of[b] % 64
        cache.k[last, :, at:], cache.v[last, :, at:] = 127, -128
    cache.upload()
    np.testing.assert_array_equal(attend(cache, bt, q, 0.125), want)


def test_attention_odd_queries():
    """A query with NaN or infinities spoils its own row and head only; huge and tiny ones stay exact to their size;
    zero scales are zero values."""
    rng = np.random.default_rng(12)
    for rows_of, len_of in (([1] * 6, [60] * 6), ([40], [90])):
        bt, cache, q = make(rng, rows_of, len_of, 32, 8, 2, 64)
        q[0, 1, 3], q[1, 5, 0], q[2, 7] = np.nan, np.inf, 0
        q[3] *= np.float32(1e-30)
        q[4, 2] *= np.float32(1e20)
        cache.vs[bt.table[0, 0]] = 0
        cache.ks[bt.table[0, 1], 0] = 0
        cache.vs[bt.table[-1, 1]] *= np.float32(1e-12)
        cache.upload()
        want = np.full(q.shape, 7.25)
        tol = ref.attention(q, *bt.plain(), cache.k, cache.v, cache.ks, cache.vs, 0.125, 0, want)
        got = attend(cache, bt, q, 0.125)
        np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
        fine = ~np.isnan(want)
        tol[4, 2] = np.inf                                  # scores of 1e20: a softmax of one, compared below
        assert np.all(np.abs(got - want)[fine] <= np.broadcast_to(tol[..., None], want.shape)[fine])
        np.testing.assert_allclose(got[4, 2], want[4, 2], rtol=0, atol=np.abs(want[4, 2]).max() * 64 * 2.0 ** -24)


def test_attention_scale_signs_and_sizes():
    rng = np.random.default_rng(13)
    bt, cache, q = make(rng, [1, 20], [50, 70], 32, 4, 2, 64)
    for scale in (0.0, -0.3, 1e-6, 4.0):
        check_attention(cache, bt, q, scale)


def test_attention_repeats_bit_for_bit():
    rng = np.random.default_rng(14)
    for rows_of, len_of in (([1] * 5, [900, 3, 77, 2000, 1024]), ([100, 33], [700, 33])):
        bt, cache, q = make(rng, rows_of, len_of, 64, 14, 2, 64)
        np.testing.assert_array_equal(attend(cache, bt, q, 0.125), attend(cache, bt, q, 0.125))
