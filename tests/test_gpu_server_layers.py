"""Whole steps of a server, every layer by itself: attention with each layer's window and sinks, the weights that it leaves, of cut
requests too, and the tokens that stay, over many steps with evictions, drafts and rewinds; and the decoder's window, from the queries
and pages that its last layer holds. Against the plain restatements of keep_ref.py, in 64 bits."""
import numpy as np
import pytest

import keep_ref as ref
import rehip
import serving_ref
from rehip import hip, qwen
from test_gpu_attention_sinks import near
from test_gpu_kv8 import Cache, i32
from test_gpu_long_conversations import (D, FIRST, GEOM, HD, HEADS, KEEP, KV, LD, LIMIT, PAGE, PAGES, RECENT, STEPS, VOCAB, Server,
                                         get)

pytestmark = pytest.mark.gpu
B = hip.DeviceBuffer
LAYERS = [(70, 4), (0, 0), (20, 40), (33, 0)]       # window and sinks: one behind the other, none, sinks past the window, no sinks


class Layers(Server):
    """A server whose layers have buffers of their own, so that a step can be looked at layer by layer afterwards."""

    def __init__(self, n, cap, seed):
        super().__init__(n, cap, seed)
        more = len(LAYERS) - len(self.caches)
        self.caches += [Cache(self.rng, PAGES, KV, PAGE, HD) for _ in range(more)]
        self.mass += [B.from_array(np.full((PAGES, KV, PAGE), 3.0, np.float32)) for _ in range(more)]
        self.ctx = [B.from_array(np.zeros((cap, HEADS, HD), np.float32)) for _ in LAYERS]
        self.lse = [B.from_array(np.zeros((cap, HEADS), np.float32)) for _ in LAYERS]
        self.kept = [i32(np.zeros((n, KV, KEEP))) for _ in LAYERS]

    def enqueue(self, s):
        b, n, cap = self.b, self.n, self.cap
        pool = (b["table"], LD, b["free"], PAGES, b["nf"])
        rehip.kv_plan_dev(n, PAGE, b["new"], b["len"], *pool, b["len"], b["nf"], b["start"], b["count"], cap, b["seq"], b["pos"],
                          b["slot"], b["status"], s)
        rehip.kv_positions_dev(cap, b["seq"], b["pos"], n, b["dropped"], b["turn"], s)
        rehip.embed_dev(b["embed"], VOCAB, D, b["tok"], cap, b["x"], s)
        rehip.rope_rows_dev(b["x"], D, cap, HEADS + KV, HD, HD, rehip.ROPE_HALF, b["freqs"], self.mscale, b["turn"], b["x"], D, s)
        batch = (cap, n, b["start"], b["count"], b["len"], b["table"], LD, PAGE, PAGES)
        k, v = b["x"].ptr + 4 * HEADS * HD, b["x"].ptr + 4 * (HEADS + KV) * HD
        for (window, sinks), c, ctx, lse, mass in zip(LAYERS, self.caches, self.ctx, self.lse, self.mass):
            rehip.kv8_append_dev(k, D, v, D, *batch, *c.args(), KV, HD, s)
            rehip.attention_kv8_sinks_dev(b["x"], D, *batch, *c.args(), cap, LD * PAGE, HEADS, KV, HD, HD ** -0.5, window, sinks, ctx,
                                          lse, self.work, self.nb, s)
            rehip.kv8_mass_dev(b["x"], D, lse, *batch, c.kb, c.ksb, cap, LD * PAGE, HEADS, KV, HD, HD ** -0.5, window, sinks, mass, s)
        self.head.matmul_dev(self.ctx[-1], cap, b["logits"], rehip.MODE_F32, s)
        rehip.draft_verify_dev(b["logits"], VOCAB, cap, VOCAB, n, b["vstart"], b["vcount"], b["tok"], None, 0, b["t"], b["u"], b["r"],
                               b["acc"], b["back"], b["out"], self.vwork, self.nv, s)
        rehip.kv_rewind_dev(n, PAGE, b["back"], b["len"], *pool, b["len"], b["nf"], s)
        rehip.kv_evict_plan_dev(n, PAGE, LIMIT, KEEP, b["len"], *pool, b["len"], b["table"], b["free"], b["nf"], b["from_len"],
                                b["old"], b["dropped"], b["status"], s)
        for c, mass, kept in zip(self.caches, self.mass, self.kept):
            rehip.kv8_evict_dev(n, b["from_len"], b["old"], b["table"], LD, PAGE, PAGES, *c.args(), mass, KV, HD, KEEP, FIRST, RECENT,
                                LD * PAGE, kept, s)

    def step_layers(self, new, go):
        """Feeds and steps with `go`; then every layer's attention, weights and move. Returns the requests that were cut."""
        self.feed(new)
        p, b, n, cap = self.state(), self.b, self.n, self.cap
        caches = [[x.copy() for x in (c.k, c.v, c.ks, c.vs)] for c in self.caches]
        before = [get(m, PAGES, KV, PAGE, dtype=np.float32) for m in self.mass]
        go()
        hip.synchronize()
        want = serving_ref.plan(PAGE, np.asarray(new), p["len"], p["table"], p["free"], int(p["nf"][0]), cap)
        batch, live = (want["start"], want["count"], want["len"], p["table"], PAGE), want["seq"] >= 0
        gx = get(b["x"], cap, HEADS + 2 * KV, HD, dtype=np.float32)
        stack = p["free"].copy()
        length, free = ref.rewind(PAGE, get(b["back"], n), want["len"], p["table"], stack, want["n_free"], PAGES)
        stack[:len(free)] = free
        left = length
        length, table, free, from_len, rows, _ = ref.evict_plan(PAGE, LIMIT, KEEP, left, p["table"], stack, len(free), None)
        np.testing.assert_array_equal(get(b["len"], n), length)
        np.testing.assert_array_equal(get(b["table"], n, LD), table)
        for (window, sinks), c, pages, had, ctx, lse, mass, kept in zip(LAYERS, caches, self.caches, before, self.ctx, self.lse,
                                                                        self.mass, self.kept):
            serving_ref.append(gx[:, HEADS:HEADS + KV], *batch, c[0], c[2])
            serving_ref.append(gx[:, HEADS + KV:], *batch, c[1], c[3])
            x, y = np.zeros((cap, HEADS, HD)), np.zeros((cap, HEADS))
            tol, tol_lse = ref.attention(gx[:, :HEADS], batch, c, HD ** -0.5, window, sinks, x, y)
            got_lse = get(lse, cap, HEADS, dtype=np.float32)
            near(get(ctx, cap, HEADS, HD, dtype=np.float32)[live], x[live], np.broadcast_to(tol[..., None], x.shape)[live])
            near(got_lse[live], y[live], tol_lse[live])
            # the masses on the pages of what each request had before the cut: a cut one's still hold them
            m = had.astype(np.float64)
            tol = ref.mass(gx[:, :HEADS], got_lse, batch, c[0], c[2], HD ** -0.5, window, sinks, m)
            got = get(mass, PAGES, KV, PAGE, dtype=np.float32)
            for i in range(n):
                used = p["table"][i, :-(-int(left[i]) // PAGE)]
                assert np.all(np.abs(got[used] - m[used]) <= tol[used]), (i, window, sinks)
            # the move, from the masses that the device has, bit by bit
            moved, stay = got.copy(), np.zeros((n, KV, KEEP), np.int32)
            ref.evict(from_len, rows, table, PAGE, c, moved, KEEP, FIRST, RECENT, stay)
            cut = from_len > 0
            np.testing.assert_array_equal(get(kept, n, KV, KEEP)[cut], stay[cut])
            np.testing.assert_array_equal(got, moved)
            pages.k, pages.v, pages.ks, pages.vs = c
            pages.check()
        return int(cut.sum())


def test_every_layer_of_a_server():
    sv = Layers(4, 150, 21)
    assert sum(sv.step_layers(new, lambda: sv.enqueue(None)) for new in STEPS) >= 1


def test_every_layer_of_a_replayed_step():
    sv, other = Layers(4, 150, 22), Layers(4, 150, 23)
    stream = hip.Stream()
    sv.head.matmul_dev(sv.ctx[-1], sv.cap, sv.b["logits"], rehip.MODE_F32, stream)    # (its partials are allocated here)
    hip.synchronize()
    graph = hip.Graph(stream, lambda: sv.enqueue(stream))
    cut = 0
    for new in STEPS:
        cut += sv.step_layers(new, lambda: (hip.synchronize(), graph.launch(), stream.synchronize()))
        other.step_layers(new, lambda: other.enqueue(None))
    assert cut >= 1
    graph.destroy()
    stream.destroy()


@pytest.mark.parametrize("use_graph", [True, False])
@pytest.mark.parametrize("window,sinks", [(40, 3), (1, 0), (17, 100), (1000, 4), (0, 0)])
def test_the_decoders_window(window, sinks, use_graph):
    """After a prompt in two chunks, steps over page borders and a drafted step: the context of the last layer's rows is that of its
    rotated queries over its pages, with this window and these sinks."""
    mb = qwen.synth_model(7, GEOM, n_layers=2, n_vocab=1000)
    rng = np.random.default_rng(5)
    dd = qwen.DeviceDecoder(mb, max_seq=300, prefill_rows=128, kv_cache="int8", window=window, sinks=sinks, use_graph=use_graph)
    g, kv, hd = dd.g, dd.g.n_kv_heads, dd.g.head_dim
    d, page, count = g.d_model, dd.pages.PAGE, dd.pages.count

    def look(rows, length):
        dd.stream.synchronize()
        q = dd.qkv.download(np.float32, rows * (d + 2 * kv * hd)).reshape(rows, -1)[:, :d].reshape(rows, g.n_heads, hd)
        kc, vc, ks, vs = dd.blocks[-1]["cache"]
        codes = [serving_ref.unpack(x.download(np.int8, count * kv * page * hd), count, kv, page, hd, i) for i, x in enumerate((kc, vc))]
        scales = [x.download(np.float32, count * kv).reshape(count, kv) for x in (ks, vs)]
        table = get(dd.pages.table, 1, count)
        batch = (np.array([0]), np.array([rows]), np.array([length]), table, page)
        ctx, lse = np.zeros(q.shape), np.zeros(q.shape[:2])
        tol, _ = ref.attention(q, batch, (*codes, *scales), hd ** -0.5, window, sinks, ctx, lse)
        near(dd.ctx.download(np.float32, rows * d).reshape(q.shape), ctx, np.broadcast_to(tol[..., None], q.shape))
    dd.prefill(rng.integers(0, 1000, 100))
    look(100, 100)
    dd.prefill(rng.integers(0, 1000, 70))
    look(70, 170)
    for i in range(30):
        dd.step()
        if i % 7 == 0 or i > 25:
            look(1, 171 + i)
    dd.step_drafted([5, 6, 7])
    look(4, 204)                        # (rows that were taken back are still what the pass computed)
    dd.close()
