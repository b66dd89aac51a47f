"""A batched serving step end to end: plan, rotary positions, append, attention and log probabilities over several steps
of a small attention model, eagerly and as one captured graph per step shape, on two streams at once, against the plain
restatements of serving_ref.py."""
import threading

import numpy as np
import pytest

import rehip
import serving_ref as ref
from rehip import hip

pytestmark = pytest.mark.gpu
B = hip.DeviceBuffer
HEADS, KV, HD, PAGE, LD, PAGES, VOCAB, TOP = 6, 2, 64, 32, 6, 18, 700, 5
D = (HEADS + 2 * KV) * HD


def i32(a):
    return B.from_array(np.ascontiguousarray(a, np.int32))


class Server:
    """Device state of up to n requests; `embed` gives a token's fused q|k|v row, `head` the logits of a context row."""

    def __init__(self, n, cap, seed):
        rng = np.random.default_rng(seed)
        self.n, self.cap = n, cap
        self.embed = rng.standard_normal((VOCAB, D)).astype(np.float32)
        w = (rng.standard_normal((VOCAB, HEADS * HD)) / 8).astype(np.float32)
        self.w = w
        self.head = rehip.QMat.from_f32(w, VOCAB, HEADS * HD)
        self.freqs, self.mscale = rehip.rope_freqs(1e4, 32, rehip.ROPE_BANDS, 4.0, 64.0)
        self.table_b = B.from_array(self.embed)
        self.freqs_b = B.from_array(self.freqs)
        self.new, self.len, self.nfree = i32(np.zeros(n)), i32(np.zeros(n)), i32([PAGES])
        self.table = i32(np.full((n, LD), -1))
        self.free = i32(np.arange(PAGES)[::-1])
        self.start, self.count, self.status = i32(np.zeros(n)), i32(np.zeros(n)), i32(np.zeros(2))
        self.seq, self.pos, self.slot = (i32(np.zeros(cap)) for _ in range(3))
        self.tok, self.targets = i32(np.zeros(cap)), i32(np.zeros(cap))
        self.x, self.ctx = B(cap * D * 4), B(cap * HEADS * HD * 4)
        self.logits = B(cap * VOCAB * 4)
        size = PAGES * KV * PAGE * HD
        self.kc, self.vc = (B.from_array(rng.integers(-128, 128, size).astype(np.int8)) for _ in range(2))
        self.ks, self.vs = (B.from_array(np.full(PAGES * KV, 3.0, np.float32)) for _ in range(2))
        self.lp, self.en = B(cap * 4), B(cap * 4)
        self.ids, self.top = B(cap * TOP * 4), B(cap * TOP * 4)
        self.work_bytes = max(rehip.attention_kv8_work_bytes(cap, n, cap, LD * PAGE, HEADS, KV, HD),
                              rehip.logprobs_work_bytes(cap, VOCAB, TOP), 16)
        self.work = B(self.work_bytes)
        # the same state, stepped plainly
        self.p = {"len": np.zeros(n, np.int32), "table": np.full((n, LD), -1, np.int32),
                  "free": np.arange(PAGES, dtype=np.int32)[::-1].copy(), "nf": PAGES,
                  "k": ref.unpack(self.kc.download(np.int8), PAGES, KV, PAGE, HD, 0),
                  "v": ref.unpack(self.vc.download(np.int8), PAGES, KV, PAGE, HD, 1),
                  "ks": np.full((PAGES, KV), 3.0, np.float32), "vs": np.full((PAGES, KV), 3.0, np.float32)}

    def enqueue(self, stream):
        """One step of `cap` rows; everything it needs to know lies in device memory."""
        s, cap, n = stream, self.cap, self.n
        rehip.kv_plan_dev(n, PAGE, self.new, self.len, self.table, LD, self.free, PAGES, self.nfree, self.len, self.nfree,
                          self.start, self.count, cap, self.seq, self.pos, self.slot, self.status, s)
        rehip.embed_dev(self.table_b, VOCAB, D, self.tok, cap, self.x, s)
        # q and k lie side by side: one call turns both
        rehip.rope_rows_dev(self.x, D, cap, HEADS + KV, HD, 32, rehip.ROPE_INTERLEAVED, self.freqs_b, self.mscale,
                            self.pos, self.x, D, s)
        batch = (cap, n, self.start, self.count, self.len, self.table, LD, PAGE, PAGES, self.kc, self.vc, self.ks, self.vs)
        k, v = self.x.ptr + 4 * HEADS * HD, self.x.ptr + 4 * (HEADS + KV) * HD
        rehip.kv8_append_dev(k, D, v, D, *batch, KV, HD, s)
        rehip.attention_kv8_dev(self.x, D, *batch, cap, LD * PAGE, HEADS, KV, HD, HD ** -0.5, 0, self.ctx, self.work,
                                self.work_bytes, s)
        self.head.matmul_dev(self.ctx, cap, self.logits, rehip.MODE_F32, s)
        rehip.logprobs_dev(self.logits, VOCAB, cap, VOCAB, self.targets, TOP, self.lp, self.en, self.ids, self.top,
                           self.work, self.work_bytes, s)

    def feed(self, rng, new):
        """The step's inputs: tokens and targets of its packed rows."""
        total = int(np.maximum(new, 0).sum())
        tok, tgt = np.full(self.cap, -1, np.int32), np.full(self.cap, -1, np.int32)
        tok[:total], tgt[:total] = rng.integers(0, VOCAB, total), rng.integers(0, VOCAB, total)
        self.new.upload(np.asarray(new, np.int32))
        self.tok.upload(tok)
        self.targets.upload(tgt)
        self.ctx.upload(np.full((self.cap, HEADS * HD), 0.5, np.float32))
        return tok, tgt

    def check(self, new, tok, tgt):
        """Device state and outputs after a step against the plain ones."""
        p, cap = self.p, self.cap
        want = ref.plan(PAGE, np.asarray(new), p["len"], p["table"], p["free"], p["nf"], cap)
        p["len"], p["nf"] = want["len"], want["n_free"]
        hip.synchronize()
        got = lambda b, t, *shape: b.download(t, int(np.prod(shape))).reshape(shape)  # noqa: E731
        np.testing.assert_array_equal(got(self.len, np.int32, self.n), p["len"])
        np.testing.assert_array_equal(got(self.table, np.int32, self.n, LD), p["table"])
        np.testing.assert_array_equal(got(self.slot, np.int32, cap), want["slot"])
        assert got(self.nfree, np.int32, 1)[0] == p["nf"] and got(self.status, np.int32, 2).tolist() == want["status"]
        x = np.where((tok >= 0)[:, None], self.embed[np.maximum(tok, 0)], 0).astype(np.float32)
        turned = ref.rope(x[:, :(HEADS + KV) * HD].reshape(cap, -1, HD), want["pos"], self.freqs, self.mscale, 32, True)
        gx = got(self.x, np.float32, cap, HEADS + 2 * KV, HD)
        # 12 roundings of terms of at most |x0| + |x1| (see test_gpu_serve_ops.py)
        np.testing.assert_allclose(gx[:, :HEADS + KV], turned, rtol=0, atol=12 * 2.0 ** -24 * 3 * np.abs(x).max())
        # (append and attention from what the device has turned: they are then defined bit by bit / to their own bound)
        batch = (want["start"], want["count"], p["len"], p["table"], PAGE)
        ref.append(gx[:, HEADS:HEADS + KV], *batch, p["k"], p["ks"])
        ref.append(gx[:, HEADS + KV:], *batch, p["v"], p["vs"])
        np.testing.assert_array_equal(ref.unpack(got(self.kc, np.int8, PAGES * KV * PAGE * HD), PAGES, KV, PAGE, HD, 0), p["k"])
        np.testing.assert_array_equal(ref.unpack(got(self.vc, np.int8, PAGES * KV * PAGE * HD), PAGES, KV, PAGE, HD, 1), p["v"])
        np.testing.assert_array_equal(got(self.ks, np.float32, PAGES, KV), p["ks"])
        ctx = np.full((cap, HEADS, HD), 0.5)
        tol = ref.attention(gx[:, :HEADS], *batch, p["k"], p["v"], p["ks"], p["vs"], HD ** -0.5, 0, ctx)
        gc = got(self.ctx, np.float32, cap, HEADS, HD)
        assert np.all(np.abs(gc - ctx) <= tol[..., None])
        gl = got(self.logits, np.float32, cap, VOCAB)
        lp, en, ids, top = ref.logprobs(gl, tgt, TOP)
        np.testing.assert_array_equal(got(self.ids, np.int32, cap, TOP), ids)
        tol = (700 + 4 * 2 * np.abs(gl).max()) * 2.0 ** -24   # as in test_gpu_serve_ops.py
        np.testing.assert_allclose(got(self.lp, np.float32, cap), lp, rtol=0, atol=tol)
        np.testing.assert_allclose(got(self.top, np.float32, cap, TOP), top, rtol=0, atol=tol)
        np.testing.assert_allclose(got(self.en, np.float32, cap), en, rtol=0, atol=tol * 8)
        return want


# prompts, single tokens, requests that end and begin again, idle ones; once more than the pool holds
STEPS = [[40, 0, 3, 17], [1, 30, 1, 1], [1, 1, -1, 1], [-1, 1, 20, 1], [25, 1, 1, -1], [1, 1, 1, 33], [9, 20, 1, 1],
         [30, 30, 1, 1], [1, 1, 1, 1], [-1, -1, -1, -1], [60, 0, 0, 2]]


def test_steps_of_a_server():
    sv, rng, refused = Server(4, 66, 1), np.random.default_rng(1), 0
    for new in STEPS + [[1, 64, 1, 0], [1, 1, 1, 60], [1, 1, 62, 1], [0, 60, 5, 0], [0, 0, 60, 0], [60, 0, 0, 0],
                        [0, 66, 0, 0], [0, 0, 0, 66], [66, 0, 0, 0], [0, 0, 66, 0], [1, 1, 1, 63]]:
        tok, tgt = sv.feed(rng, new)
        sv.enqueue(None)
        refused += sv.check(new, tok, tgt)["status"][0]
    assert refused


def test_steps_as_a_replayed_graph():
    """One captured graph serves every step: the batch lies in device memory. Eager steps of another server run between
    the replays."""
    sv, other, rng = Server(4, 66, 2), Server(4, 66, 3), np.random.default_rng(2)
    stream = hip.Stream()
    sv.head.matmul_dev(sv.ctx, sv.cap, sv.logits, rehip.MODE_F32, stream)      # (its partials are allocated here)
    hip.synchronize()
    graph = hip.Graph(stream, lambda: sv.enqueue(stream))
    for i, new in enumerate(STEPS):
        tok, tgt = sv.feed(rng, new)
        hip.synchronize()
        graph.launch()
        stream.synchronize()
        sv.check(new, tok, tgt)
        if i % 3 == 0:
            otok, otgt = other.feed(rng, new)
            other.enqueue(None)
            other.check(new, otok, otgt)
    graph.destroy()


def test_two_servers_on_two_streams_at_once():
    """Two threads, each with its own stream and server."""
    servers, errors = [Server(4, 66, 4), Server(4, 66, 5)], []

    def work(sv, seed):
        try:
            rng, stream = np.random.default_rng(seed), hip.Stream()
            for new in STEPS:
                tok, tgt = sv.feed(rng, new)
                hip.synchronize()
                sv.enqueue(stream)
                stream.synchronize()
                sv.check(new, tok, tgt)
        except BaseException as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(sv, i)) for i, sv in enumerate(servers)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    if errors:
        raise errors[0]
