"""A server whose conversations outgrow their pages and which decodes drafted tokens: plan, positions, append, attention
with sinks, weights, eviction, verification and rewind over many steps of a small attention model, eagerly, as captured
graphs and for two servers at once, against the plain restatements. The decoder's window and drafted steps. Edges of the
new calls: pages past 32-bit offsets, many requests, shared workspaces' neighbours, misuse that is allowed."""
import threading

import numpy as np
import pytest

import keep_ref as ref
import rehip
import serving_ref
from rehip import hip, qwen
from test_gpu_attention_sinks import attend_sinks, check, check_mass, near, weigh
from test_gpu_draft_verify import drafts
from test_gpu_kv8 import Batch, Cache, i32, make

pytestmark = pytest.mark.gpu
B = hip.DeviceBuffer
HEADS, KV, HD, PAGE, LD, PAGES, VOCAB = 6, 2, 64, 32, 7, 40, 500
D = (HEADS + 2 * KV) * HD
WINDOW, SINKS, LIMIT, KEEP, FIRST, RECENT = 70, 4, 120, 90, 4, 40


def get(buf, *shape, dtype=np.int32):
    return buf.download(dtype, int(np.prod(shape))).reshape(shape)


class Server:
    """Up to n requests with up to `most` drafts each; two layers' caches share one plan, and only the second one's masses
    differ from the first's."""

    def __init__(self, n, cap, seed):
        rng = self.rng = np.random.default_rng(seed)
        self.n, self.cap = n, cap
        self.embed = rng.standard_normal((VOCAB, D)).astype(np.float32)
        self.head = rehip.QMat.from_f32((rng.standard_normal((VOCAB, HEADS * HD)) / 2).astype(np.float32), VOCAB, HEADS * HD)
        self.freqs, self.mscale = rehip.rope_freqs(1e4, HD)
        self.b = dict(embed=B.from_array(self.embed), freqs=B.from_array(self.freqs), new=i32(np.zeros(n)), len=i32(np.zeros(n)),
                      nf=i32([PAGES]), table=i32(np.full((n, LD), -1)), old=i32(np.full((n, LD), -1)), free=i32(np.arange(PAGES)[::-1]),
                      start=i32(np.zeros(n)), count=i32(np.zeros(n)), status=i32([0, 0]), from_len=i32(np.zeros(n)),
                      dropped=i32(np.zeros(n)), vstart=i32(np.zeros(n)), vcount=i32(np.zeros(n)), acc=i32(np.zeros(n)), back=i32(np.zeros(n)), out=i32(np.zeros(cap)),
                      seq=i32(np.zeros(cap)), pos=i32(np.zeros(cap)), slot=i32(np.zeros(cap)), turn=i32(np.zeros(cap)),
                      tok=i32(np.zeros(cap)), t=B.from_array(np.array([0.7, 0, 1.2, 1], np.float32)[np.arange(n) % 4]),
                      u=B(cap * 4), r=B(n * 4), x=B(cap * D * 4), ctx=B.from_array(np.zeros((cap, HEADS * HD), np.float32)),
                      lse=B.from_array(np.zeros((cap, HEADS), np.float32)), logits=B(cap * VOCAB * 4),
                      kept=i32(np.zeros((n, KV, KEEP))))
        self.caches = [Cache(rng, PAGES, KV, PAGE, HD) for _ in range(2)]
        self.mass = [B.from_array(np.full((PAGES, KV, PAGE), 3.0, np.float32)) for _ in range(2)]
        self.nb = max(rehip.attention_kv8_work_bytes(cap, n, cap, LD * PAGE, HEADS, KV, HD), 16)
        self.nv = rehip.draft_verify_work_bytes(cap, n, VOCAB)
        self.work, self.vwork = B(self.nb), B(self.nv)

    def enqueue(self, s):
        """One step of `cap` rows; everything it needs to know lies in device memory."""
        b, n, cap = self.b, self.n, self.cap
        pool = (b["table"], LD, b["free"], PAGES, b["nf"])
        rehip.kv_plan_dev(n, PAGE, b["new"], b["len"], *pool, b["len"], b["nf"], b["start"], b["count"], cap, b["seq"], b["pos"],
                          b["slot"], b["status"], s)
        rehip.kv_positions_dev(cap, b["seq"], b["pos"], n, b["dropped"], b["turn"], s)
        rehip.embed_dev(b["embed"], VOCAB, D, b["tok"], cap, b["x"], s)
        rehip.rope_rows_dev(b["x"], D, cap, HEADS + KV, HD, HD, rehip.ROPE_HALF, b["freqs"], self.mscale, b["turn"], b["x"], D, s)
        batch = (cap, n, b["start"], b["count"], b["len"], b["table"], LD, PAGE, PAGES)
        k, v = b["x"].ptr + 4 * HEADS * HD, b["x"].ptr + 4 * (HEADS + KV) * HD
        for layer, c in enumerate(self.caches):
            rehip.kv8_append_dev(k, D, v, D, *batch, *c.args(), KV, HD, s)
            window = (WINDOW, SINKS) if layer == 0 else (0, 0)
            rehip.attention_kv8_sinks_dev(b["x"], D, *batch, *c.args(), cap, LD * PAGE, HEADS, KV, HD, HD ** -0.5, *window,
                                          b["ctx"], b["lse"], self.work, self.nb, s)
            rehip.kv8_mass_dev(b["x"], D, b["lse"], *batch, c.kb, c.ksb, cap, LD * PAGE, HEADS, KV, HD, HD ** -0.5, *window,
                               self.mass[layer], s)
        self.head.matmul_dev(b["ctx"], cap, b["logits"], rehip.MODE_F32, s)
        rehip.draft_verify_dev(b["logits"], VOCAB, cap, VOCAB, n, b["vstart"], b["vcount"], b["tok"], None, 0, b["t"], b["u"], b["r"],
                               b["acc"], b["back"], b["out"], self.vwork, self.nv, s)
        rehip.kv_rewind_dev(n, PAGE, b["back"], b["len"], *pool, b["len"], b["nf"], s)
        rehip.kv_evict_plan_dev(n, PAGE, LIMIT, KEEP, b["len"], *pool, b["len"], b["table"], b["free"], b["nf"], b["from_len"],
                                b["old"], b["dropped"], b["status"], s)
        for layer, c in enumerate(self.caches):
            rehip.kv8_evict_dev(n, b["from_len"], b["old"], b["table"], LD, PAGE, PAGES, *c.args(), self.mass[layer], KV, HD, KEEP,
                                FIRST, RECENT, LD * PAGE, b["kept"], s)

    def feed(self, new):
        """The step's inputs. Up to five new tokens are the last one and drafts, of more (a prompt) the last row alone draws."""
        rng, b, p = self.rng, self.b, self.state()
        plan = serving_ref.plan(PAGE, np.asarray(new), p["len"], p["table"], p["free"], int(p["nf"][0]), self.cap)
        count = np.where(plan["count"] > 5, 1, plan["count"])
        b["vcount"].upload(count.astype(np.int32))
        b["vstart"].upload((plan["start"] + plan["count"] - count).astype(np.int32))
        b["new"].upload(np.asarray(new, np.int32))
        tok = np.full(self.cap, -1, np.int32)
        total = int(np.maximum(new, 0).sum())
        tok[:total] = rng.integers(0, VOCAB, total)
        b["tok"].upload(tok)
        b["u"].upload(rng.random(self.cap).astype(np.float32) * np.float32(0.02))       # (random drafts: some are accepted)
        b["r"].upload(rng.random(self.n).astype(np.float32))
        b["ctx"].upload(np.zeros((self.cap, HEADS * HD), np.float32))
        b["out"].upload(np.full(self.cap, -7, np.int32))

    def state(self):
        b = self.b
        return {k: get(b[k], *s) for k, s in (("len", (self.n,)), ("table", (self.n, LD)), ("free", (PAGES,)), ("nf", (1,)),
                                              ("dropped", (self.n,)))}

    def step_checked(self, new, go):
        """Feeds and steps with `go`, the outcome against the plain one from the state before."""
        self.feed(new)
        p, b, n, cap = self.state(), self.b, self.n, self.cap
        caches = [[x.copy() for x in (c.k, c.v, c.ks, c.vs)] for c in self.caches]
        masses = [get(m, PAGES, KV, PAGE, dtype=np.float32) for m in self.mass]
        go()
        hip.synchronize()
        want = serving_ref.plan(PAGE, np.asarray(new), p["len"], p["table"], p["free"], int(p["nf"][0]), cap)
        turn = np.where(want["seq"] >= 0, want["pos"] + p["dropped"][want["seq"]], -1)
        np.testing.assert_array_equal(get(b["turn"], cap), turn)
        tok = get(b["tok"], cap)
        x = np.where((tok >= 0)[:, None], self.embed[np.maximum(tok, 0)], 0).reshape(cap, -1, HD)
        gx = get(b["x"], cap, HEADS + 2 * KV, HD, dtype=np.float32)
        # 12 roundings of terms of at most |x0| + |x1| (see test_gpu_serve_ops.py)
        np.testing.assert_allclose(gx[:, :HEADS + KV], serving_ref.rope(x[:, :HEADS + KV], turn, self.freqs, self.mscale, HD, False),
                                   rtol=0, atol=12 * ref.EPS * 3 * np.abs(x).max())
        batch = (want["start"], want["count"], want["len"], p["table"], PAGE)
        logits = get(b["logits"], cap, VOCAB, dtype=np.float32)
        for layer, c in enumerate(caches):
            serving_ref.append(gx[:, HEADS:HEADS + KV], *batch, c[0], c[2])
            serving_ref.append(gx[:, HEADS + KV:], *batch, c[1], c[3])
        # the second layer's attention is what the device holds
        ctx, lse = np.zeros((cap, HEADS, HD)), np.zeros((cap, HEADS))
        tol, tol_lse = ref.attention(gx[:, :HEADS], batch, caches[1], HD ** -0.5, 0, 0, ctx, lse)
        live = want["seq"] >= 0
        near(get(b["ctx"], cap, HEADS, HD, dtype=np.float32)[live], ctx[live], np.broadcast_to(tol[..., None], ctx.shape)[live])
        glse = get(b["lse"], cap, HEADS, dtype=np.float32)
        near(glse[live], lse[live], tol_lse[live])
        tokens = np.full(cap, -7, np.int32)
        acc, back = ref.verify(logits, get(b["vstart"], n), get(b["vcount"], n), tok, None, get(b["t"], n, dtype=np.float32),
                               get(b["u"], cap, dtype=np.float32), get(b["r"], n, dtype=np.float32), tokens)
        np.testing.assert_array_equal(get(b["acc"], n), acc)
        np.testing.assert_array_equal(get(b["out"], cap), tokens)
        stack = p["free"].copy()
        length, free = ref.rewind(PAGE, back, want["len"], p["table"], stack, want["n_free"], PAGES)
        stack[:len(free)] = free
        length, table, free, from_len, rows, _ = ref.evict_plan(PAGE, LIMIT, KEEP, length, p["table"], stack, len(free), p["dropped"])
        after = self.state()
        np.testing.assert_array_equal(after["len"], length)
        np.testing.assert_array_equal(after["table"], table)
        np.testing.assert_array_equal(after["free"][:len(free)], free)
        np.testing.assert_array_equal(after["dropped"], p["dropped"])
        assert after["nf"][0] == len(free)
        # the first layer's masses to their bound (its lse is what a second, equal call gives), the second's by the lse at hand; then
        # the move, bit by bit, from the device's masses
        for layer, c in enumerate(caches):
            got = get(self.mass[layer], PAGES, KV, PAGE, dtype=np.float32)
            if layer == 1:
                m = masses[1].astype(np.float64)
                tol = ref.mass(gx[:, :HEADS], glse, batch, c[0], c[2], HD ** -0.5, 0, 0, m)
                for i in range(n):
                    if from_len[i] == 0:
                        used = p["table"][i, :-(-length[i] // PAGE)]
                        assert np.all(np.abs(got[used] - m[used]) <= tol[used])
            kept, dk = np.zeros((n, KV, KEEP), np.int32), get(b["kept"], n, KV, KEEP)
            old = [x.copy() for x in c]
            # (a cut request's masses before the move are gone from the new pages alone: the old ones still hold them)
            moved = got.copy()
            ref.evict(from_len, rows, table, PAGE, c, moved, KEEP, FIRST, RECENT, kept)
            cut = from_len > 0
            if layer == 1:
                np.testing.assert_array_equal(dk[cut], kept[cut])
            np.testing.assert_array_equal(got, moved)
            for i in range(4):
                np.testing.assert_array_equal((lambda d: serving_ref.unpack(d, PAGES, KV, PAGE, HD, i) if i < 2 else d.reshape(PAGES, KV))(
                    (self.caches[layer].kb, self.caches[layer].vb, self.caches[layer].ksb, self.caches[layer].vsb)[i].download(
                        np.int8 if i < 2 else np.float32, old[i].size)), c[i])
            self.caches[layer].k, self.caches[layer].v, self.caches[layer].ks, self.caches[layer].vs = c
        return {"cut": int((from_len > 0).sum()), "accepted": int(acc.sum()), "back": int(back.sum())}


STEPS = [[100, 0, 30, 17], [1, 60, 5, 1], [5, 5, 4, 1], [5, 5, -1, 5], [3, 5, 110, 5], [5, 5, 5, 5], [5, -1, 5, 90], [5, 20, 3, 5],
         [5, 5, 5, 5], [5, 1, 5, 5], [-1, 80, 5, 5], [0, 30, 5, 5], [115, 5, 5, 5], [5, 5, 5, 5], [5, 5, 5, 5]]


def test_steps_of_a_server():
    sv, seen = Server(4, 150, 1), {"cut": 0, "accepted": 0, "back": 0}
    for new in STEPS:
        for k, v in sv.step_checked(new, lambda: sv.enqueue(None)).items():
            seen[k] += v
    assert seen["cut"] >= 2 and seen["accepted"] > 0 and seen["back"] > 20


def test_steps_as_a_replayed_graph():
    """One captured graph serves every step; eager steps of another server run between the replays."""
    sv, other = Server(4, 150, 2), Server(4, 150, 3)
    stream = hip.Stream()
    sv.head.matmul_dev(sv.b["ctx"], sv.cap, sv.b["logits"], rehip.MODE_F32, stream)   # (its partials are allocated here)
    hip.synchronize()
    graph = hip.Graph(stream, lambda: sv.enqueue(stream))
    cut = 0
    for new in STEPS:
        cut += sv.step_checked(new, lambda: (hip.synchronize(), graph.launch(), stream.synchronize()))["cut"]
        other.step_checked(new, lambda: other.enqueue(None))
    assert cut >= 2
    graph.destroy()
    stream.destroy()


def test_two_servers_at_once():
    """Each with its own stream, buffers and workspaces, their steps overlapping."""
    servers, errors = [Server(4, 150, s) for s in (4, 5)], []

    def work(sv):
        try:
            stream = hip.Stream()
            for new in STEPS:
                sv.step_checked(new, lambda: (sv.enqueue(stream), stream.synchronize()))
            stream.destroy()
        except BaseException as e:       # noqa: B036 (handed to the main thread)
            errors.append(e)
    threads = [threading.Thread(target=work, args=(sv,)) for sv in servers]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    if errors:
        raise errors[0]


# ---- edges ---------------------------------------------------------------------------------------
def test_pages_past_32_bit_offsets():
    """Pages whose codes lie behind 2^32 bytes: attention, weights and the move of tokens there and back."""
    page, hd, kv, heads = 256, 256, 16, 16
    n_pages = (1 << 32) // (page * hd * kv) + 3
    rng = np.random.default_rng(1)
    far = np.array([n_pages - 1, n_pages - 2], np.int32)
    bt = Batch(rng, [1], [400], page, spare=0, ld_extra=0)
    bt.table[0] = far
    bt.n_pages = n_pages
    small = Cache(rng, 2, kv, page, hd)
    small.ks, small.vs = (np.full((2, kv), 0.01, np.float32) for _ in range(2))
    size = page * hd * kv

    class Far:
        shape = (n_pages, kv, page, hd)
        kb, vb = B(n_pages * size), B(n_pages * size)
        ksb, vsb = B.from_array(np.zeros((n_pages, kv), np.float32)), B.from_array(np.zeros((n_pages, kv), np.float32))

        def args(self):
            return self.kb, self.vb, self.ksb, self.vsb
    f = Far()
    put = lambda buf, at, a: hip.check(hip.hip().hipMemcpy(buf.ptr + at, a.ctypes.data, a.nbytes, hip.H2D))  # noqa: E731
    for i, p in enumerate(far):
        for buf, codes, v in ((f.kb, small.k, 0), (f.vb, small.v, 1)):
            put(buf, int(p) * size, np.ascontiguousarray(serving_ref.pack(codes[i:i + 1], v)))
        for buf, sc in ((f.ksb, small.ks), (f.vsb, small.vs)):
            put(buf, int(p) * kv * 4, np.ascontiguousarray(sc[i]))
    q = rng.standard_normal((1, heads, hd)).astype(np.float32)
    near_table = bt.table.copy()
    near_table[0] = [0, 1]
    for window, sinks in ((0, 0), (100, 4)):
        ctx, lse = np.zeros(q.shape), np.zeros(q.shape[:2])
        batch = (bt.start, bt.count, bt.len, near_table, page)
        tol, tol_lse = ref.attention(q, batch, (small.k, small.v, small.ks, small.vs), 1 / 16, window, sinks, ctx, lse)
        got, got_lse = attend_sinks(f, bt, q, 1 / 16, window, sinks)
        near(got, ctx, np.broadcast_to(tol[..., None], q.shape))
        near(got_lse, lse, tol_lse)
    mb = B.from_array(np.zeros((n_pages, kv, page), np.float32))
    rehip.kv8_mass_dev(B.from_array(q), heads * hd, B.from_array(got_lse), *bt.args(), f.kb, f.ksb, 1, 400, heads, kv, hd, 1 / 16, 100,
                       4, mb)
    hip.synchronize()
    want = np.zeros((2, kv, page))
    tol = ref.mass(q, got_lse, (bt.start, bt.count, bt.len, near_table, page), small.k, small.ks, 1 / 16, 100, 4, want)
    got = mb.download(np.float32).reshape(n_pages, kv, page)[far]
    assert np.all(np.abs(got - want) <= tol)
    # from the far pages to a near one
    kept = i32(np.zeros((kv, 200)))
    to = np.array([[0, -1]], np.int32)
    rehip.kv8_evict_dev(1, i32([400]), i32(bt.table), i32(to), 2, page, n_pages, *f.args(), mb, kv, hd, 200, 4, 150, 400, kept)
    hip.synchronize()
    k = get(kept, kv, 200)
    code = lambda buf, v: serving_ref.unpack(buf.download(np.int8, size), 1, kv, page, hd, v)[0]  # noqa: E731
    gk, gv = code(f.kb, 0), code(f.vb, 1)
    for h in range(kv):
        m = got[:, h].reshape(-1)[:400].astype(np.float64)
        order = sorted(range(4, 250), key=lambda t: (-m[t], t))[:46]
        np.testing.assert_array_equal(k[h], np.sort(np.r_[np.arange(4), order, np.arange(250, 400)]))
        np.testing.assert_array_equal(gk[h, :200], small.k[k[h] // page, h, k[h] % page])
        np.testing.assert_array_equal(gv[h, :200], small.v[k[h] // page, h, k[h] % page])


@pytest.mark.parametrize("requests,most,rows", [(65, 300, 1), (300, 150, 1), (1024, 40, 2), (1500, 60, 1), (1500, 30, 3)])
def test_masses_of_many_requests(requests, most, rows):
    """Pieces found by a lane each, from a list, and in even chunks."""
    rng = np.random.default_rng(requests)
    len_of = rng.integers(0, most + 1, requests)
    len_of[requests // 2] = 700
    bt, cache, q = make(rng, np.minimum(len_of, rng.integers(0, rows + 1, requests)), len_of, 32, 4, 2, 32)
    check_mass(cache, bt, q, 0.2, 0, 0, max_rows=max(int(bt.count.max()), 1), max_len=most)


def test_masses_of_prompts_of_many_requests():
    rng = np.random.default_rng(2)
    bt, cache, q = make(rng, rng.integers(0, 40, 70), 40 + rng.integers(0, 60, 70), 32, 8, 2, 32)
    check_mass(cache, bt, q, 0.2, 20, 2)
    bt, cache, q = make(rng, [40] * 1100, [41 + i % 50 for i in range(1100)], 32, 4, 2, 32)
    check_mass(cache, bt, q, 0.2, 0, 0)


@pytest.mark.parametrize("hd,kv_heads,page", [(32, 4, 32), (64, 2, 64), (96, 2, 32), (128, 3, 96), (160, 1, 32), (256, 2, 64)])
@pytest.mark.parametrize("requests,window,sinks", [(2, 0, 0), (2, 37, 5), (60, 0, 0), (60, 37, 5), (130, 20, 2)])
def test_masses_by_shares_of_waves(hd, kv_heads, page, requests, window, sinks):
    """Steps whose pieces are shared by two waves (many requests of a few rows), four and eight (long prompts of few)."""
    rng = np.random.default_rng(hd + requests)
    few, grp = requests == 2, 8
    rows = [150, 97] if few else rng.integers(0, 14, requests)
    len_of = np.array([400, 97]) if few else np.minimum(rng.integers(0, 120, requests) + rows, 120)
    bt, cache, q = make(rng, rows, len_of, page, grp * kv_heads, kv_heads, hd)
    most = int(np.max(rows))
    assert (grp * most >= 1024) if few else 64 < grp * most <= 256
    for max_len in (400, 8000):                                    # (four waves at the second)
        check_mass(cache, bt, q, hd ** -0.5, window, sinks, max_rows=most, max_len=max_len if few else 40 * max_len // 2)


def test_starts_that_do_not_ascend_stay_in_bounds():
    """Rubbish in the batch arrays: nothing is read or written out of place (what comes out is not looked at)."""
    rng = np.random.default_rng(3)
    bt, cache, q = make(rng, [5, 3, 9], [40, 70, 33], 32, 8, 2, 64)
    for start, count, length in (([9, 0, 4], [5, 3, 9], [40, 70, 33]), ([-5, 1 << 30, 3], [1 << 30, -4, 9], [1 << 30, -7, 33]),
                                 ([0, 0, 0], [17, 17, 17], [10, 1 << 20, 5])):
        bt.start, bt.count, bt.len = (np.array(a, np.int32) for a in (start, count, length))
        _, lse = attend_sinks(cache, bt, q, 0.1, 20, 4, max_rows=9, max_len=70)
        weigh(cache, bt, q, np.zeros_like(lse), 0.1, 20, 4, np.zeros(cache.shape[:3]), max_rows=9, max_len=70)
        x, _, _, tokens, p, u, r = drafts(rng, [6, 6, 5], 50)
        nb = rehip.draft_verify_work_bytes(17, 3, 50)
        o = [i32(np.zeros(3)), i32(np.zeros(3)), i32(np.zeros(17))]
        rehip.draft_verify_dev(B.from_array(x), 50, 17, 50, 3, i32(start), i32(count), i32(tokens), B.from_array(p), 50, None,
                               B.from_array(u), B.from_array(r), *o, B.from_array(np.zeros(nb, np.uint8)), nb)
    hip.synchronize()


def test_an_idle_pool():
    """Nothing over the limit, nothing to take back: everything is left as it was."""
    rng = np.random.default_rng(4)
    cache = Cache(rng, 9, 2, 32, 64)
    table = i32(np.arange(8).reshape(2, 4))
    mass, kept = B.from_array(np.ones((9, 2, 32), np.float32)), i32(np.full((2, 2, 50), -3))
    rehip.kv8_evict_dev(2, i32([0, 0]), i32(np.full((2, 4), 5)), table, 4, 32, 9, *cache.args(), mass, 2, 64, 50, 4, 4, 128, kept)
    cache.check()
    assert np.all(get(kept, 200) == -3) and np.all(get(mass, 576, dtype=np.float32) == 1)


# ---- the decoder -----------------------------------------------------------------------------------
GEOM = qwen.Geometry(d_model=256, n_heads=4, n_kv_heads=2, d_ff=512, rope_freq_base=1e4, rms_eps=1e-5)


@pytest.fixture(scope="module")
def tiny():
    return qwen.synth_model(7, GEOM, n_layers=3, n_vocab=1000)


def test_decoder_windows_are_checked(tiny):
    for bad in ({"window": 9}, {"sinks": 2}, {"window": -1, "kv_cache": "int8"}, {"window": 9, "sinks": 1025, "kv_cache": "int8"}):
        with pytest.raises(ValueError):
            qwen.DeviceDecoder(tiny, max_seq=100, prefill_rows=50, **bad)


def test_decoder_with_a_window(tiny):
    """A window longer than the sequence changes nothing but the order of no sum; a short one, prompt by chunks or at once, graph
    or not, gives the same tokens, and other logits than the whole sequence."""
    prompt = np.random.default_rng(1).integers(0, 1000, 150)
    got = {}
    for name, k in {"whole": {}, "wide": dict(window=1000, sinks=4), "short": dict(window=40, sinks=3),
                    "eager": dict(window=40, sinks=3, use_graph=False)}.items():
        dd = qwen.DeviceDecoder(tiny, max_seq=400, prefill_rows=200, kv_cache="int8", **k)
        tokens = [dd.prefill(prompt)] + [dd.step() for _ in range(20)]
        got[name] = tokens, dd.logits()
        dd.close()
    assert got["wide"][0] == got["whole"][0] and got["short"][0] == got["eager"][0]
    np.testing.assert_array_equal(got["wide"][1], got["whole"][1])
    np.testing.assert_array_equal(got["short"][1], got["eager"][1])
    assert not np.array_equal(got["short"][1], got["whole"][1])


@pytest.mark.parametrize("kv_cache", ["f32", "int8"])
def test_drafted_steps(tiny, kv_cache):
    """Drafts that are the greedy tokens are accepted, others are not, and the sequence goes on as if only the accepted had been
    decoded: tokens, position, history and, to the gate that the int8 pages pass, logits."""
    prompt = np.random.default_rng(3).integers(0, 1000, 100)
    plain = qwen.DeviceDecoder(tiny, max_seq=400, prefill_rows=200, kv_cache=kv_cache)
    want, lg = [plain.prefill(prompt)], []
    for _ in range(30):
        want.append(plain.step())
        lg.append(plain.logits())
    dd = qwen.DeviceDecoder(tiny, max_seq=400, prefill_rows=200, kv_cache=kv_cache)
    assert dd.prefill(prompt) == want[0]
    at = 0
    for good, bad in ((4, 0), (0, 1), (2, 3), (0, 0), (7, 1), (3, 2)):
        offered = want[at + 1:at + 1 + good] + [(want[at + 1 + good] + 1 + i) % 1000 for i in range(bad)]
        got = dd.step_drafted(offered)
        assert got == want[at + 1:at + 2 + good] and dd.seq_len == 100 + at + 1 + good
        at += good + 1
        gate = qwen.logit_profile_check(lg[at - 1], dd.logits())
        assert gate["ok"], (at, gate)
    assert dd.history(100, at + 1) == want[:at + 1]
    assert dd.step() == want[at + 1]                            # (and single steps go on from there)
    for bad in ([1000], [-1], [0] * 300):
        with pytest.raises(ValueError):
            dd.step_drafted(bad)
    with pytest.raises(ValueError):
        dd.step_drafted([1], temperature=1.0)
    assert dd.seq_len == 100 + at + 1
    tokens = dd.step_drafted([5, 6], temperature=0.8, accept_u=[0.0, 0.0], sample_u=0.5)      # (0: accepted with any weight)
    assert tokens[:2] == [5, 6] and len(tokens) == 3
    q = np.full((2, 1000), 1e-3, np.float32)
    assert 1 <= len(dd.step_drafted([5, 6], temperature=0.8, probs=q, accept_u=[0.5, 0.5], sample_u=0.25)) <= 3
    dd.close()
    dd = qwen.DeviceDecoder(tiny, max_seq=400, prefill_rows=200, kv_cache=kv_cache)
    assert dd.generate_drafted(prompt, 31) == want
    dd.close()
    plain.close()


def test_drafted_steps_of_growing_length(tiny):
    """The buffers of a step grow with its drafts and serve shorter ones afterwards; a sequence that is full ends them."""
    prompt = np.random.default_rng(4).integers(0, 1000, 20)
    plain = qwen.DeviceDecoder(tiny, max_seq=50, prefill_rows=32, kv_cache="int8")
    want = [plain.prefill(prompt)] + [plain.step() for _ in range(30)]
    plain.close()
    dd = qwen.DeviceDecoder(tiny, max_seq=50, prefill_rows=32, kv_cache="int8")
    assert dd.prefill(prompt) == want[0]
    at = 0
    for n in (1, 6, 2, 0, 9):
        assert dd.step_drafted(want[at + 1:at + 1 + n]) == want[at + 1:at + 2 + n]
        at += n + 1
    with pytest.raises(ValueError):
        dd.step_drafted(want[:7])                               # (seven drafts and the token before them: one place too few)
    assert dd.step_drafted(want[at + 1:at + 7]) == want[at + 1:at + 8] and dd.seq_len == 50
    assert dd.history(20, 30) == want[:30]                       # (the token behind the last place is in no history)
    dd.close()


def test_lookup_drafts():
    assert qwen.lookup_drafts([1, 2, 3, 4, 1, 2], 4) == [3, 4, 1, 2]
    assert qwen.lookup_drafts([1, 2, 3, 1, 2, 5, 1, 2], 1) == [5]
    assert qwen.lookup_drafts([1, 2, 3], 4) == [] and qwen.lookup_drafts([1, 2], 4) == [] and qwen.lookup_drafts([1, 1, 1], 0) == []
