"""Eviction from the paged int8 cache (plan and move, bit for bit) and tokens taken back, against the plain restatements of
keep_ref.py."""
import numpy as np
import pytest

import keep_ref as ref
import rehip
import serving_ref
from rehip import hip
from test_gpu_kv8 import Cache, i32

pytestmark = pytest.mark.gpu
B = hip.DeviceBuffer


def get(buf, n, dtype=np.int32):
    hip.synchronize()
    return buf.download(dtype, n)


class Pool:
    """Requests of given lengths in shuffled pages, `spare` free ones."""

    def __init__(self, rng, len_of, page, spare, ld_extra=1):
        self.len = np.asarray(len_of, np.int32)
        need = -(-self.len // page)
        self.n, self.page, self.ld = len(len_of), page, int(need.max()) + ld_extra
        self.n_pages = int(need.sum()) + spare
        order = rng.permutation(self.n_pages).astype(np.int32)
        self.table = np.full((self.n, self.ld), -1, np.int32)
        self.table[np.arange(self.ld)[None] < need[:, None]] = order[:need.sum()]
        self.free = np.full(self.n_pages, -9, np.int32)
        self.n_free = spare
        self.free[:spare] = order[need.sum():]
        self.dropped = rng.integers(0, 50, self.n).astype(np.int32)


def run_plan(p, limit, keep, in_place, dropped=True):
    """The library's plan: (lengths, table, stack, height, from_len, old rows, dropped, status)."""
    n, ld = p.n, p.ld
    d = dict(len=i32(p.len), table=i32(p.table), free=i32(p.free), nf=i32([p.n_free]), dropped=i32(p.dropped))
    new = d if in_place else dict(len=i32(np.full(n, -5)), table=i32(np.full((n, ld), -5)),
                                  free=i32(np.full(p.n_pages, -5)), nf=i32([-5]))
    from_len, status = i32(np.full(n, -5)), i32([-5, -5])
    from_table = i32(np.full((n, ld), -5)) if in_place else d["table"]
    rehip.kv_evict_plan_dev(n, p.page, limit, keep, d["len"], d["table"], ld, d["free"], p.n_pages, d["nf"], new["len"],
                            new["table"], new["free"], new["nf"], from_len, from_table, d["dropped"] if dropped else None,
                            status)
    if not in_place:                     # the inputs are left
        np.testing.assert_array_equal(get(d["len"], n), p.len)
        np.testing.assert_array_equal(get(d["table"], n * ld).reshape(n, ld), p.table)
        np.testing.assert_array_equal(get(d["free"], p.n_pages), p.free)
    return dict(len=get(new["len"], n), table=get(new["table"], n * ld).reshape(n, ld), free=get(new["free"], p.n_pages),
                n_free=int(get(new["nf"], 1)[0]), from_len=get(from_len, n), rows=get(from_table, n * ld).reshape(n, ld),
                dropped=get(d["dropped"], n), status=get(status, 2).tolist(),
                bufs=dict(new, from_len=from_len, from_table=from_table))


def check_plan(p, limit, keep, in_place):
    dropped = p.dropped.copy()
    want = ref.evict_plan(p.page, limit, keep, p.len, p.table, p.free, p.n_free, dropped)
    got = run_plan(p, limit, keep, in_place)
    np.testing.assert_array_equal(got["len"], want[0])
    np.testing.assert_array_equal(got["table"], want[1])
    assert got["n_free"] == len(want[2]) and got["status"] == want[5]
    np.testing.assert_array_equal(got["free"][:got["n_free"]], want[2])
    np.testing.assert_array_equal(got["from_len"], want[3])
    np.testing.assert_array_equal(got["dropped"], dropped)
    for b, row in want[4].items():
        held = -(-int(want[3][b]) // p.page)
        np.testing.assert_array_equal(got["rows"][b, :held], row[:held])
    return got, want


LENGTHS = {
    "one": [300],
    "some": [0, 64, 65, 200, 1, 63, 300, 128],
    "none": [3, 0, 50],
    "all": [130 + 17 * i for i in range(20)],
}


@pytest.mark.parametrize("name", LENGTHS)
@pytest.mark.parametrize("page,limit,keep,spare", [(32, 100, 40, 50), (32, 64, 64, 9), (64, 100, 1, 2), (16, 129, 127, 20),
                                                   (32, 100, 100, 0)])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan(name, page, limit, keep, spare, in_place):
    """Requests over and under the limit, pages for all, some and none of them, the outputs in place and not."""
    rng = np.random.default_rng(page + limit + spare)
    check_plan(Pool(rng, LENGTHS[name], page, spare), limit, keep, in_place)


@pytest.mark.parametrize("n,ld_extra", [(256, 0), (257, 90), (1024, 0), (1025, 3), (4096, 2)])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan_of_many_requests(n, ld_extra, in_place):
    rng = np.random.default_rng(n)
    p = Pool(rng, rng.integers(0, 90, n), 8, 3 * n, ld_extra)
    got, want = check_plan(p, 50, 37, in_place)
    assert want[5][1] > n // 4
    p = Pool(rng, rng.integers(0, 90, n), 8, n // 2, ld_extra)
    _, want = check_plan(p, 50, 37, in_place)
    assert want[5][0] > 0


def test_plan_of_unsound_lengths():
    """Lengths outside the table are left; entries that hold no page are not given back; a garbage stack count."""
    rng = np.random.default_rng(3)
    p = Pool(rng, [200, 200, 200, 200], 32, 12)
    p.len[0], p.len[2] = -3, p.ld * 32 + 1
    p.table[1, 1], p.table[1, 3], p.table[3, 0] = -1, p.n_pages, 1 << 30
    check_plan(p, 100, 60, False)
    check_plan(p, 100, 60, True)
    p.n_free = -4
    got = run_plan(p, 100, 60, False)
    assert got["n_free"] == 0 and got["status"] == [2, 0]
    assert run_plan(p, 100, 60, False, dropped=False)["dropped"].tolist() == p.dropped.tolist()


# ---- the move --------------------------------------------------------------------------------------
def check_evict(rng, len_of, page, kv_heads, hd, limit, keep, first, recent, spare=60, masses="some", spoil=None, max_len=None):
    p = Pool(rng, len_of, page, spare)
    if spoil:
        spoil(p)
    cache = Cache(rng, p.n_pages, kv_heads, page, hd)
    m = np.round(4 * rng.standard_normal((p.n_pages, kv_heads, page))).astype(np.float32) / 4     # (ties, negative ones)
    if masses == "odd":
        m[rng.random(m.shape) < 0.2] = np.nan
        m[rng.random(m.shape) < 0.1] = np.inf
        m[rng.random(m.shape) < 0.1] = -np.inf
    if masses == "equal":
        m[:] = 0.5
    if masses == "fine":
        m = np.exp(rng.standard_normal(m.shape)).astype(np.float32)
    if masses is None:
        m = None
    got, want = check_plan(p, limit, keep, False)
    kept = np.full((p.n, kv_heads, keep), -7, np.int32)
    mb, kb, d = None if m is None else B.from_array(m), i32(kept), got["bufs"]
    rehip.kv8_evict_dev(p.n, d["from_len"], d["from_table"], d["table"], p.ld, page, p.n_pages, *cache.args(), mb, kv_heads, hd,
                        keep, first, recent, int(max(p.len.max(), 1)) if max_len is None else max_len, kb)
    ref.evict(want[3], want[4], want[1], page, (cache.k, cache.v, cache.ks, cache.vs), m, keep, first, recent, kept)
    np.testing.assert_array_equal(get(kb, kept.size).reshape(kept.shape), kept)
    cache.check()
    if m is not None:
        np.testing.assert_array_equal(get(mb, m.size, np.float32).reshape(m.shape), m)
    return kept


@pytest.mark.parametrize("page,hd,kv_heads", [(32, 64, 2), (64, 128, 3), (64, 32, 1), (96, 96, 2), (128, 160, 1),
                                              (256, 256, 2)])
@pytest.mark.parametrize("limit,keep,first,recent", [(100, 70, 4, 20), (200, 1, 0, 0), (150, 150, 0, 150), (130, 64, 64, 0),
                                                     (256, 129, 1, 31)])
def test_evict(page, hd, kv_heads, limit, keep, first, recent):
    rng = np.random.default_rng(page + hd + keep)
    check_evict(rng, [120, 50, 300, 517, 0, 151], page, kv_heads, hd, limit, keep, first, recent)


@pytest.mark.parametrize("masses", ["odd", "equal", "fine", None])
def test_evict_of_odd_masses(masses):
    """NaN and infinities, all equal (the earliest stay), and none at all (the first and the last stay)."""
    rng = np.random.default_rng(11)
    kept = check_evict(rng, [700, 90, 333], 32, 2, 64, 300, 200, 8, 192 if masses is None else 60, masses=masses)
    if masses == "equal":
        np.testing.assert_array_equal(kept[0, 0], np.r_[0:140, 640:700])


@pytest.mark.parametrize("len_of,keep,first,recent,max_len", [([16500], 8000, 4, 100, None), ([40000, 300], 39999, 0, 0, None),
                                                              ([33000], 500, 0, 17, 100), ([17000], 16999, 500, 115, None)])
def test_evict_of_long_requests(len_of, keep, first, recent, max_len):
    """More tokens than a workgroup holds at a time; longer than planned."""
    rng = np.random.default_rng(keep)
    check_evict(rng, len_of, 64, 1, 32, keep, keep, first, recent, spare=700, masses="fine", max_len=max_len)


@pytest.mark.parametrize("keep,first,recent", [(90, 40, 50), (90, 90, 0), (90, 0, 90), (33, 1, 32)])
def test_evict_to_the_ends(keep, first, recent):
    """Nothing to pick: absent pages among the old ones, lengths that nothing is cut of, masses that move along."""
    def spoil(p):
        p.table[0, 1], p.table[0, 3], p.table[1] = -1, p.n_pages + 3, -1
        p.len[2] = p.ld * p.page + 1
    check_evict(np.random.default_rng(keep + first), [300, 200, 250, 500, 20, 100, 101], 32, 2, 64, 100, keep, first, recent, spoil=spoil)


def test_evict_with_absent_pages():
    """Tokens without a page are the first to go; those that stay have code, scale and mass 0."""
    def spoil(p):
        p.table[0, 1], p.table[0, 3], p.table[1] = -1, p.n_pages + 3, -1
        p.len[2] = p.ld * p.page + 1
    check_evict(np.random.default_rng(12), [300, 200, 250, 500], 32, 2, 64, 100, 90, 40, 20, spoil=spoil)
    check_evict(np.random.default_rng(13), [300, 200, 250, 500], 32, 2, 64, 100, 99, 0, 0, spoil=spoil, masses="odd")


def test_evict_leaves_what_attention_sees():
    """Only tokens of no weight go: attention after the cut is attention before it, but for the codes' rounding to the new
    pages' scales (half a step of at most the old page's, so less than 1 / 254 of the largest value in each operand)."""
    rng = np.random.default_rng(14)
    page, hd, h = 32, 64, 1
    p = Pool(rng, [400], page, 20)
    cache = Cache(rng, p.n_pages, h, page, hd)
    cache.ks[:], cache.vs[:] = 0.02, 0.02            # one scale: nothing is rounded
    m = np.zeros((p.n_pages, h, page), np.float32)
    heavy = np.sort(rng.choice(400, 100, replace=False))
    for t in range(400):
        if t not in heavy:
            cache.k[p.table[0, t // page], 0, t % page] = -127
        m[p.table[0, t // page], 0, t % page] = t in heavy
    cache.upload()
    q = np.full((1, 1, hd), 1.0, np.float32)          # sees tokens of -127 with e^-20 of the weight at most
    cache.k[p.table[0, heavy // page], 0, heavy % page] = np.abs(cache.k[p.table[0, heavy // page], 0, heavy % page].astype(int)).clip(0, 127)
    cache.upload()
    def attend(length, table):
        work = rehip.attention_kv8_work_bytes(1, 1, 1, 400, 1, 1, hd)
        ctx = B.from_array(np.zeros(hd, np.float32))
        rehip.attention_kv8_dev(B.from_array(q), hd, 1, 1, i32([0]), i32([1]), length, table, p.ld, page, p.n_pages,
                                *cache.args(), 1, 400, 1, 1, hd, 0.25, 0, ctx, B(max(work, 16)), work)
        return get(ctx, hd, np.float32)
    before = attend(i32(p.len), i32(p.table))
    got = run_plan(p, 200, 100, False)
    d = got["bufs"]
    rehip.kv8_evict_dev(1, d["from_len"], d["from_table"], d["table"], p.ld, page, p.n_pages, *cache.args(), B.from_array(m), h,
                        hd, 100, 0, 0, 400, i32(np.zeros(100)))
    after = attend(d["len"], d["table"])
    # scores of the light tokens are below the heavy ones' mean by 0.25 * 64 * 0.02 * 127 = 40: e^-40 of 300 of them, and
    # both sides' f32 arithmetic (keep_ref.attention's bound at 400 tokens: scores up to 41)
    np.testing.assert_allclose(after, before, rtol=0, atol=2.54 * (4 * 80 * 2.0 ** -24 * 41 + 2 * 89 * 2.0 ** -24))


# ---- rewind --------------------------------------------------------------------------------------
def check_rewind(p, back, in_place=False):
    want_len, want_free = ref.rewind(p.page, back, p.len, p.table, p.free, max(min(p.n_free, p.n_pages), 0), p.n_pages)
    ln, nf = i32(p.len), i32([p.n_free])
    lo, no = (ln, nf) if in_place else (i32(np.full(p.n, -5)), i32([-5]))
    table, free = i32(p.table), i32(p.free)
    rehip.kv_rewind_dev(p.n, p.page, i32(back), ln, table, p.ld, free, p.n_pages, nf, lo, no)
    np.testing.assert_array_equal(get(lo, p.n), want_len)
    n_free = int(get(no, 1)[0])
    assert n_free == len(want_free)
    np.testing.assert_array_equal(get(free, p.n_pages)[:n_free], want_free)
    np.testing.assert_array_equal(get(table, p.n * p.ld).reshape(p.n, p.ld), p.table)
    return want_len, want_free


@pytest.mark.parametrize("n,page,most,back", [(1, 64, 300, 5), (7, 32, 200, 40), (64, 64, 8192, 4), (256, 16, 100, 16), (257, 8, 60, 60),
                                              (1024, 16, 90, 16), (1500, 1, 20, 20), (4096, 16, 100, 16)])
@pytest.mark.parametrize("in_place", [False, True])
def test_rewind(n, page, most, back, in_place):
    rng = np.random.default_rng(n)
    p = Pool(rng, rng.integers(0, most + 1, n), page, 5)
    check_rewind(p, rng.integers(-2, back + 1, n).astype(np.int32), in_place)
    check_rewind(p, np.full(n, 1 << 30, np.int32), in_place)       # all of it
    check_rewind(p, np.zeros(n, np.int32), in_place)


def test_rewind_of_unsound_lengths():
    rng = np.random.default_rng(4)
    p = Pool(rng, [200, 200, 200, 200, 1], 32, 3)
    p.len[0], p.len[2] = -3, p.ld * 32 + 1
    p.table[1, 5], p.table[1, 6], p.table[3, 6] = -1, p.n_pages, 1 << 30
    check_rewind(p, np.array([9, 150, 9, 50, -(1 << 31)], np.int32))
    p.n_free = -7
    check_rewind(p, np.array([9, 150, 9, 50, 1], np.int32))
    p.n_free = p.n_pages + 9                                    # a full stack takes no more
    ln = i32(p.len)
    nf, free = i32([p.n_free]), i32(np.arange(p.n_pages))
    rehip.kv_rewind_dev(p.n, 32, i32([9] * 5), ln, i32(p.table), p.ld, free, p.n_pages, nf, ln, nf)
    assert get(nf, 1)[0] == p.n_pages and get(free, p.n_pages).tolist() == list(range(p.n_pages))


def test_rewind_and_plan_go_on():
    """Steps of drafts, some taken back: every page has one owner or is free, as if the rejected rows had never been."""
    rng = np.random.default_rng(5)
    n, page, ld, pages = 9, 8, 12, 80
    kv_len, table, free, nf = i32(np.zeros(n)), i32(np.full((n, ld), -1)), i32(rng.permutation(pages)), i32([pages])
    o = [i32(np.zeros(n)) for _ in range(2)] + [i32(np.zeros(200)) for _ in range(3)] + [i32([0, 0])]
    length = np.zeros(n, int)
    for _ in range(30):
        new = rng.integers(1, 10, n)
        new[rng.random(n) < 0.1] = -1
        rehip.kv_plan_dev(n, page, i32(new), kv_len, table, ld, free, pages, nf, kv_len, nf, o[0], o[1], 200, *o[2:5], o[5])
        count = get(o[1], n)
        back = np.where(count > 0, rng.integers(0, 10, n) % np.maximum(count, 1), 0)
        rehip.kv_rewind_dev(n, page, i32(back), kv_len, table, ld, free, pages, nf, kv_len, nf)
        length = np.where(new < 0, 0, length + count - back)
        np.testing.assert_array_equal(get(kv_len, n), length)
        t = get(table, n * ld).reshape(n, ld)
        used = [t[b, :-(-length[b] // page)] for b in range(n)] + [get(free, pages)[:get(nf, 1)[0]]]
        assert sorted(np.concatenate(used)) == list(range(pages))


def test_evict_rounds_the_rounded_product():
    """Codes whose product with the ratio of scales is next to half a code: the product is rounded to f32 before it is rounded
    to a code, so those that f32 takes to the half go to the even one."""
    page, hd, n = 32, 64, 120
    c = np.arange(1, 128)
    ratios, hits = [], 0
    for k in range(n):                   # (k + 1/2) / c of some c above k, rounded: c times it is next to k + 1/2
        code = int(c[c > k][k * 7 % (127 - k)])
        r = np.float32((k + 0.5) / code)
        ratios.append(r)
        exact = float(r) * code
        hits += np.rint(np.float32(code) * r) != np.rint(exact)
    assert hits > 10
    p = Pool(np.random.default_rng(15), [64] * n, page, n + 1)
    cache = Cache(np.random.default_rng(16), p.n_pages, 1, page, hd)
    for b in range(n):                   # one page of this scale, one of scale 1, tokens of both in the new one
        cache.ks[p.table[b, :2], 0] = cache.vs[p.table[b, :2], 0] = ratios[b], 1.0
        for codes in (cache.k, cache.v):
            codes[p.table[b, 0], 0] = np.arange(-64, 64)[None].repeat(16, 0).reshape(page, hd) if b % 2 else np.arange(
                64, 128)[None].repeat(page, 0)
    cache.upload()
    got, want = check_plan(p, 40, 32, False)
    d, kept = got["bufs"], np.zeros((n, 1, 32), np.int32)
    rehip.kv8_evict_dev(n, d["from_len"], d["from_table"], d["table"], p.ld, page, p.n_pages, *cache.args(), None, 1, hd, 32, 31, 1, 64,
                        i32(kept))
    ref.evict(want[3], want[4], want[1], page, (cache.k, cache.v, cache.ks, cache.vs), None, 32, 31, 1, kept)
    cache.check()
