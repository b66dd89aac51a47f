"""The plan of a batched step, rotary positions of a batch's rows and log probabilities, against the plain
restatements of serving_ref.py."""
import numpy as np
import pytest

import rehip
import serving_ref as ref
from rehip import hip

pytestmark = pytest.mark.gpu
B = hip.DeviceBuffer
EPS = 2.0 ** -24                 # half a step of f32, relative


def i32(a):
    return B.from_array(np.ascontiguousarray(a, np.int32))


def get(buf, n, dtype=np.float32):
    hip.synchronize()
    return buf.download(dtype, n)


# ---- plan --------------------------------------------------------------------------------------
class Pool:
    """Requests' state on the device and beside it the same state stepped by the plain plan."""

    def __init__(self, requests, page, ld, n_pages, rng):
        self.n, self.page, self.ld, self.n_pages = requests, page, ld, n_pages
        self.len = np.zeros(requests, np.int32)
        self.table = np.full((requests, ld), -7, np.int32)
        self.free = rng.permutation(n_pages).astype(np.int32)
        self.n_free = n_pages
        self.dev = {"len": i32(self.len), "table": i32(self.table), "free": i32(self.free), "nf": i32([n_pages])}

    def step(self, new, cap, alias=True):
        d, n = self.dev, self.n
        o = {k: i32(np.full(max(m, 1), -5)) for k, m in (("start", n), ("count", n), ("seq", cap), ("pos", cap),
                                                         ("slot", cap), ("status", 2), ("len", n), ("nf", 1))}
        lo, nfo = (d["len"], d["nf"]) if alias else (o["len"], o["nf"])
        rehip.kv_plan_dev(n, self.page, i32(new), d["len"], d["table"], self.ld, d["free"], self.n_pages, d["nf"], lo,
                          nfo, o["start"], o["count"], cap, o["seq"], o["pos"], o["slot"], o["status"])
        want = ref.plan(self.page, np.asarray(new), self.len, self.table, self.free, self.n_free, cap)
        for k in ("start", "count"):
            np.testing.assert_array_equal(get(o[k], n, np.int32), want[k], k)
        for k in ("seq", "pos", "slot"):
            np.testing.assert_array_equal(get(o[k], cap, np.int32), want[k], k)
        np.testing.assert_array_equal(get(lo, n, np.int32), want["len"])
        assert get(nfo, 1, np.int32)[0] == want["n_free"]
        assert get(o["status"], 2, np.int32).tolist() == want["status"]
        np.testing.assert_array_equal(get(d["table"], n * self.ld, np.int32).reshape(n, -1), self.table)
        np.testing.assert_array_equal(get(d["free"], self.n_pages, np.int32), self.free)
        if not alias:
            np.testing.assert_array_equal(get(d["len"], n, np.int32), self.len)    # inputs are left
        self.len, self.n_free = want["len"], want["n_free"]
        self.dev.update(len=lo, nf=nfo)
        return want


@pytest.mark.parametrize("requests,page,ld,n_pages,most", [(1, 64, 1, 1, 64), (1, 1, 9, 5, 3), (7, 32, 6, 20, 70),
                                                           (64, 64, 8, 200, 40), (64, 64, 8, 70, 40), (1000, 16, 5, 3000, 30),
                                                           (4096, 8, 3, 5000, 9)])
def test_plan_steps(requests, page, ld, n_pages, most):
    """Steps of a pool: requests grow, end, begin again and are refused, for want of pages or of table room."""
    rng = np.random.default_rng(requests + page)
    p = Pool(requests, page, ld, n_pages, rng)
    refused = 0
    for step in range(8):
        new = rng.integers(0, most + 1, requests)
        new[rng.random(requests) < 0.15] = -1
        total = int(np.maximum(new, 0).sum())
        cap = [total, total + 7, max(total - 3, 0), 0][step % 4]
        refused += p.step(new, cap, alias=step % 3 != 1)["status"][0]
    assert refused or n_pages in (1, 200)                    # (those two pools are large enough)
    held = -(-p.len // page)
    used = np.concatenate([p.table[b, :held[b]] for b in range(requests)] + [p.free[:p.n_free]])
    assert sorted(used) == list(range(n_pages))              # every page has one owner or is free


def test_plan_of_unsound_lengths():
    """Lengths and counts outside the table, a garbage stack count: refused, nothing out of place."""
    rng = np.random.default_rng(3)
    p = Pool(6, 32, 4, 16, rng)
    p.step([5, 40, 3, 3, 3, 3], 60)
    bad = p.len.copy()
    bad[1], bad[2] = -9, 1 << 30
    d, o = p.dev, [i32(np.full(6, -5)) for _ in range(6)]
    new = np.array([1, 1, 1, 1 << 30, 129, -5], np.int32)
    rows = [i32(np.full(8, -5)) for _ in range(3)]
    rehip.kv_plan_dev(6, 32, i32(new), i32(bad), d["table"], 4, d["free"], 16, i32([1 << 29]), o[0], o[1], o[2], o[3],
                      8, *rows, o[4])
    assert get(o[3], 6, np.int32).tolist() == [1, 0, 0, 0, 0, 0]
    assert get(o[0], 6, np.int32).tolist() == [6, -9, 1 << 30, 3, 3, 0]
    assert get(rows[0], 8, np.int32).tolist() == [0] + [-1] * 7
    np.testing.assert_array_equal(get(d["table"], 24, np.int32).reshape(6, 4), p.table)


# ---- rotary positions --------------------------------------------------------------------------
@pytest.mark.parametrize("rows,heads,hd,rot,extra", [(1, 1, 2, 2, 0), (3, 16, 64, 64, 0), (5, 3, 96, 24, 8),
                                                     (2, 36, 128, 64, 4), (7, 5, 256, 256, 3), (9, 2, 80, 80, 0),
                                                     (130, 18, 64, 32, 64), (4, 7, 50, 22, 1), (3, 9, 36, 36, 12)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_rows(rows, heads, hd, rot, extra, interleaved):
    """Whole and partial heads, strided rows, far positions, rows without one, in place and not."""
    rng = np.random.default_rng(rows * 100 + hd + rot)
    ld = heads * hd + extra
    x = rng.standard_normal((rows, ld)).astype(np.float32)
    pos = rng.integers(0, 1 << 20, rows).astype(np.int32)
    pos[0] = 0
    if rows > 2:
        pos[1] = -1
    freqs, mscale = rehip.rope_freqs(1e6, rot, rehip.ROPE_YARN if rot > 2 else rehip.ROPE_NONE, 8.0, 4096.0)
    want = ref.rope(x[:, :heads * hd].reshape(rows, heads, hd), pos, freqs, mscale, rot, interleaved)
    layout = rehip.ROPE_INTERLEAVED if interleaved else rehip.ROPE_HALF
    # cos and sin: the angle's reduction to f32 (2^-24 turns of pi: 4 EPS), the functions (2 ulp: 4 EPS), mscale, then
    # two products and a sum: 12 roundings in all of terms of at most |x0| + |x1|
    size = np.abs(want).max() + np.abs(x).max() * 2 * mscale
    tol = 12 * EPS * size
    for ldo in (ld, heads * hd + 5):
        out = B.from_array(np.full((rows, ldo), 7.0, np.float32))
        rehip.rope_rows_dev(B.from_array(x), ld, rows, heads, hd, rot, layout, B.from_array(freqs), mscale, i32(pos),
                            out, ldo)
        got = get(out, rows * ldo).reshape(rows, ldo)
        live = pos >= 0
        np.testing.assert_allclose(got[live, :heads * hd].reshape(-1, heads, hd), want[live], rtol=0, atol=tol)
        if rot < hd:
            np.testing.assert_array_equal(got[live, :heads * hd].reshape(-1, heads, hd)[..., rot:],
                                          x[live, :heads * hd].reshape(-1, heads, hd)[..., rot:])
        assert np.all(got[:, heads * hd:] == 7.0) and np.all(got[~live] == 7.0)
    xb = B.from_array(x)
    rehip.rope_rows_dev(xb, ld, rows, heads, hd, rot, layout, B.from_array(freqs), mscale, i32(pos), xb, ld)
    got = get(xb, rows * ld).reshape(rows, ld)
    np.testing.assert_allclose(got[:, :heads * hd].reshape(rows, heads, hd), want, rtol=0, atol=tol)
    np.testing.assert_array_equal(got[:, heads * hd:], x[:, heads * hd:])


def test_rope_unaligned_rows():
    """Rows at addresses that are multiples of 4 bytes only, odd strides."""
    rng = np.random.default_rng(1)
    rows, heads, hd, rot, ld = 5, 3, 64, 64, 201
    x = rng.standard_normal(rows * ld + 3).astype(np.float32)
    freqs, m = rehip.rope_freqs(1e4, rot)
    pos = np.arange(rows, dtype=np.int32) * 1000
    xb = B.from_array(x)
    at = lambda buf: buf.ptr + 4  # noqa: E731
    rehip.rope_rows_dev(at(xb), ld, rows, heads, hd, rot, rehip.ROPE_HALF, B.from_array(freqs), m, i32(pos), at(xb), ld)
    got = get(xb, x.size)
    body = np.lib.stride_tricks.as_strided(x[1:], (rows, heads, hd), (ld * 4, hd * 4, 4))
    want = ref.rope(body, pos, freqs, m, rot, False)
    for r in range(rows):
        np.testing.assert_allclose(got[1 + r * ld:1 + r * ld + heads * hd].reshape(heads, hd), want[r], rtol=0,
                                   atol=12 * EPS * 3 * np.abs(x).max())
    rest = np.ones(x.size, bool)
    for r in range(rows):
        rest[1 + r * ld:1 + r * ld + heads * hd] = False
    np.testing.assert_array_equal(got[rest], x[rest])


def test_rope_agrees_with_the_single_sequence_call():
    """Half layout, all of the head, consecutive positions: re_rope_dev's rotation (whose angles are f32:
    position 300 off by up to 300 * 2^-24 * 2 radians)."""
    rng = np.random.default_rng(2)
    x = rng.standard_normal((4, 6 * 64)).astype(np.float32)
    a, b = B.from_array(x), B.from_array(x)
    rehip.rope_dev(a, 4, 6, 64, 1e4, i32([297]))
    freqs, m = rehip.rope_freqs(1e4, 64)
    rehip.rope_rows_dev(b, 384, 4, 6, 64, 64, rehip.ROPE_HALF, B.from_array(freqs), m, i32([297, 298, 299, 300]), b, 384)
    np.testing.assert_allclose(get(b, x.size), get(a, x.size), rtol=0, atol=300 * 4 * EPS * 2 * np.abs(x).max())


# ---- log probabilities -------------------------------------------------------------------------
def run_logprobs(x, targets, k, ld=None, stream=None):
    rows, vocab = x.shape
    ld = ld or vocab
    full = np.full((rows, ld), 99.0, np.float32)           # values behind a row's end count for nothing
    full[:, :vocab] = x
    nb = rehip.logprobs_work_bytes(rows, vocab, k)
    work = B.from_array(np.full(max(nb // 4, 1), np.nan, np.float32))
    lp, en, top = (B.from_array(np.full(max(n, 1), 7.0, np.float32)) for n in (rows, rows, rows * k))
    ids = i32(np.full(max(rows * k, 1), -5))
    rehip.logprobs_dev(B.from_array(full), ld, rows, vocab, i32(targets), k, lp, en, ids if k else None,
                       top if k else None, work, nb, stream)
    return (get(lp, rows), get(en, rows), get(ids, rows * k, np.int32).reshape(rows, k),
            get(top, rows * k).reshape(rows, k))


def check_logprobs(x, targets, k, ld=None):
    got, want = run_logprobs(x, targets, k, ld), list(ref.logprobs(x, targets, k))
    with np.errstate(over="ignore"):                        # (a logit 6e38 below the largest is -inf in 32 bits)
        want[0], want[3] = (w.astype(np.float32).astype(np.float64) for w in (want[0], want[3]))
    np.testing.assert_array_equal(got[2], want[2])
    # d = x - m exact to EPS |d|; ln Z to its sum's relative error (at most 2 vocab-long chains of 600 steps and exp's
    # 2 ulp of |d| e^d ..: below 1e-4 relative at worst, 40 EPS typical) -- bounded here by chains of 700 roundings
    finite = np.where(np.isfinite(x), x, 0).astype(np.float64)
    spread = np.abs(finite).max(-1) * 2 + np.log(x.shape[1])
    tol = (700 * EPS + 4 * EPS * spread)
    for g, w in ((got[0], want[0]), (got[3], want[3])):
        np.testing.assert_array_equal(np.isnan(g), np.isnan(w))
        np.testing.assert_array_equal(g == -np.inf, w == -np.inf)
        fine = np.isfinite(w)
        t = np.broadcast_to(tol.reshape(-1, *[1] * (w.ndim - 1)), w.shape)
        assert np.all(np.abs(g[fine] - w[fine]) <= t[fine])
    np.testing.assert_array_equal(np.isnan(got[1]), np.isnan(want[1]))
    fine = np.isfinite(want[1])
    # the entropy's sum has terms d e^d / Z up to |d|, each off by the same chain
    assert np.all(np.abs(got[1] - want[1])[fine] <= (tol * (1 + np.log(x.shape[1])))[fine])
    return got


@pytest.mark.parametrize("rows,vocab,k", [(1, 1, 1), (3, 2, 2), (1, 63, 5), (2, 64, 64), (5, 65, 64), (1, 1000, 0),
                                          (7, 1023, 1), (300, 257, 20), (1, 151936, 20), (2, 151935, 64), (3, 32001, 7),
                                          (40, 32768, 20), (1025, 515, 3), (1541, 3000, 20), (1536, 1025, 64)])
def test_logprobs(rows, vocab, k):
    rng = np.random.default_rng(rows + vocab)
    x = (3 * rng.standard_normal((rows, vocab))).astype(np.float32)
    t = rng.integers(0, vocab, rows)
    if rows > 2:
        t[1], t[2] = -1, vocab
    check_logprobs(x, t, k, vocab + rng.integers(0, 6))


@pytest.mark.parametrize("vocab", [200, 5000, 70001])
def test_logprobs_of_hard_rows(vocab):
    """Equal logits (ties go to the lower id), rising and falling rows (every value a new best, or none), masks of
    -inf and of the lowest float, single survivors, rows without a distribution."""
    rng = np.random.default_rng(vocab)
    low = np.finfo(np.float32).min
    i = np.arange(vocab)
    normal = rng.standard_normal(vocab)
    rows = [np.zeros(vocab), np.full(vocab, low), np.full(vocab, -80.0), i * 1e-3, -i * 1e-3, (i % 7) * 1.0,
            np.where(i % 3 == 0, normal, -np.inf), np.where(i % 5 == 1, normal, low),
            np.where(i == vocab - 1, 2.0, -np.inf), np.where(i == 0, 2.0, -np.inf), np.where(i < 3, 1.0, -np.inf),
            np.full(vocab, -np.inf), np.where(i == 17, np.inf, normal), np.where(i == 99, np.nan, normal),
            1e4 * normal, np.where(i == 5, 3e38, -3e38), np.where(i % 2, -0.0, 0.0), np.full(vocab, np.nan)]
    x = np.stack(rows).astype(np.float32)
    t = rng.integers(0, vocab, len(rows))
    t[8], t[9] = vocab - 1, 3
    got = check_logprobs(x, t, 20)
    assert got[0][8] == 0 and got[1][8] == 0 and got[0][9] == -np.inf
    assert got[2][0].tolist() == list(range(20))
    check_logprobs(x, t, 64)
    if vocab < 6000:                                        # .. and a wave per row
        check_logprobs(np.tile(x, (90, 1)), np.tile(t, 90), 20)


def test_logprobs_parts_may_be_left_out():
    x = np.random.default_rng(0).standard_normal((4, 3001)).astype(np.float32)
    t = np.arange(4)
    want = run_logprobs(x, t, 6)
    nb = rehip.logprobs_work_bytes(4, 3001, 6)
    work = B(max(nb, 16))
    ids, top, en, lp = i32(np.zeros(24)), B(96), B(16), B(16)
    xb = B.from_array(x)
    rehip.logprobs_dev(xb, 3001, 4, 3001, None, 6, None, None, ids, top, work, nb)
    np.testing.assert_array_equal(get(ids, 24, np.int32).reshape(4, 6), want[2])
    rehip.logprobs_dev(xb, 3001, 4, 3001, None, 0, None, en, None, None, work, nb)
    rehip.logprobs_dev(xb, 3001, 4, 3001, i32(t), 0, lp, None, None, None, work, nb)
    np.testing.assert_allclose(get(en, 4), want[1], rtol=20 * EPS * 12, atol=0)
    np.testing.assert_allclose(get(lp, 4), want[0], rtol=20 * EPS * 12, atol=0)


def test_logprobs_repeat_bit_for_bit():
    x = (2 * np.random.default_rng(5).standard_normal((37, 40000))).astype(np.float32)
    a, b = (run_logprobs(x, np.arange(37), 20) for _ in range(2))
    for u, v in zip(a, b):
        np.testing.assert_array_equal(u, v)
