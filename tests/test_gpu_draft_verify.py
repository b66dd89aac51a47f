"""Drafted tokens against the target's probabilities, from given random numbers: every whole number equal to the plain
restatement of keep_ref.py in 64 bits."""
import numpy as np
import pytest

import keep_ref as ref
import rehip
from rehip import hip
from test_gpu_kv8 import i32

pytestmark = pytest.mark.gpu
B = hip.DeviceBuffer


def get(buf, n, dtype=np.int32):
    hip.synchronize()
    return buf.download(dtype, n)


def run(x, start, count, tokens, probs, temperature, u, r, ld=None, ldp=None, stream=None):
    rows, vocab = x.shape
    n = len(start)
    ld, ldp = ld or vocab, ldp or vocab

    def strided(a, width, fill):
        full = np.full((rows, width), fill, np.float32)
        full[:, :vocab] = a
        return B.from_array(full)
    nb = rehip.draft_verify_work_bytes(rows, n, vocab)
    work = B.from_array(np.full(nb, 255, np.uint8))
    acc, back, out = i32(np.full(n, -5)), i32(np.full(n, -5)), i32(np.full(rows, -5))
    f = lambda a: B.from_array(np.ascontiguousarray(a, np.float32))  # noqa: E731
    rehip.draft_verify_dev(strided(x, ld, np.inf), ld, rows, vocab, n, i32(start), i32(count), i32(tokens),
                           None if probs is None else strided(probs, ldp, np.nan), ldp,
                           None if temperature is None else f(temperature), f(u), f(r), acc, back, out, work, nb, stream)
    return get(acc, n), get(back, n), get(out, rows)


def check(x, start, count, tokens, probs, temperature, u, r, **k):
    got = run(x, start, count, tokens, probs, temperature, u, r, **k)
    out = np.full(len(x), -5, np.int32)
    acc, back = ref.verify(x, start, count, tokens, probs, temperature, u, r, out)
    np.testing.assert_array_equal(got[0], acc)
    np.testing.assert_array_equal(got[1], back)
    np.testing.assert_array_equal(got[2], out)
    return got


def drafts(rng, count, vocab, gap=0, sharp=3.0, probs=True, likely=0.8):
    """Rows of logits with a likely token each, drafts that often are it, and the draft model's probabilities."""
    count = np.asarray(count, np.int32)
    start = (np.concatenate([[0], np.cumsum(count + gap)])[:-1]).astype(np.int32)
    rows = int(start[-1] + count[-1] + gap)
    x = rng.standard_normal((rows, vocab)).astype(np.float32)
    top = rng.integers(0, vocab, rows)
    x[np.arange(rows), top] += np.float32(np.log(vocab) + sharp - 2)
    y = x + rng.standard_normal(x.shape).astype(np.float32) * 0.5
    q = np.exp(y - y.max(-1, keepdims=True))
    q = (q / q.sum(-1, keepdims=True)).astype(np.float32)
    drawn = np.where(rng.random(rows) < likely, top, rng.integers(0, vocab, rows))
    tokens = np.roll(drawn, 1).astype(np.int32)
    return x, start, count, tokens, q if probs else None, rng.random(rows).astype(np.float32), rng.random(len(count)).astype(np.float32)


COUNTS = {"one row": [1], "four drafts": [5], "ragged": [3, 1, 0, 5, 2, 0, 1], "long": [40, 2, 9], "many": [4] * 100 + [1] * 200}


@pytest.mark.parametrize("name", COUNTS)
@pytest.mark.parametrize("vocab", [1, 2, 63, 64, 1000, 4097])
@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("temperature", [None, "mixed"])
def test_verify(name, vocab, probs, temperature):
    rng = np.random.default_rng(vocab + len(COUNTS[name]) + probs)
    x, start, count, tokens, q, u, r = drafts(rng, COUNTS[name], vocab, gap=vocab % 2, probs=probs)
    t = None
    if temperature:
        t = (0.2 + rng.random(len(count))).astype(np.float32)
        t[rng.random(len(count)) < 0.3] = 0
    got = check(x, start, count, tokens, q, t, u, r, ld=vocab + 3, ldp=vocab + 5)
    assert vocab == 1 or name != "many" or (got[0].sum() > 0 and got[1].sum() > 0)     # (both kinds are there)


@pytest.mark.parametrize("rows_of,vocab", [([5], 151936), ([5, 3, 1, 4], 151936), ([1], 1 << 20), ([2] * 12, 32000)])
@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("flat", [False, True])
def test_large_vocabularies(rows_of, vocab, probs, flat):
    """Rows cut into parts; flat ones, where sums in 32 bits would draw neighbours."""
    rng = np.random.default_rng(vocab + len(rows_of))
    x, start, count, tokens, q, u, r = drafts(rng, rows_of, vocab, sharp=-20 if flat else 3.0, probs=probs)
    if flat:
        x *= np.float32(0.01)
    check(x, start, count, tokens, q, None, u, r)


def test_random_numbers_at_their_ends():
    """0 and the largest below 1, against tokens of no weight before and behind the others."""
    rng = np.random.default_rng(3)
    below1 = np.nextafter(np.float32(1), np.float32(0))
    x, start, count, tokens, q, u, r = drafts(rng, [2] * 40, 300)
    x[:, :7] = -np.inf
    x[:, -9:] = -np.inf
    q[:, :20] = 0
    for ends in ((0, 0), (0, below1), (below1, 0), (below1, below1)):
        u[:], r[:] = ends
        check(x, start, count, tokens, q, None, u, r)
        check(x, start, count, tokens, None, None, u, r)


def test_rows_without_a_distribution():
    """NaN, +inf, nothing above -inf: the draft is not accepted, the token is -1; other rows are as without them."""
    rng = np.random.default_rng(4)
    x, start, count, tokens, q, u, r = drafts(rng, [3] * 12, 200)
    u[:] = 0                             # (drafts with any weight are accepted)
    x[0, 5], x[4, 199], x[8, 0] = np.nan, np.inf, np.nan
    x[9], x[13], x[17] = -np.inf, -np.inf, -np.inf
    x[19, 3:] = -np.inf
    x[18, :] = np.nan
    x[21] = np.where(np.arange(200) == 77, 5.0, -np.inf)
    for t in (None, np.zeros(12, np.float32)):
        for probs in (q, None):
            got = check(x, start, count, tokens, probs, t, u, r)
            assert got[2][0] == -1 and got[0][0] == 0
    assert not np.any(got[2] < -1)


def test_temperatures():
    """From nearly greedy to nearly flat, infinite, negative, NaN, in one batch."""
    rng = np.random.default_rng(5)
    t = np.array([1e-30, 1e-6, 0.01, 0.5, 1, 2, 100, 1e6, 1e30, np.inf, -1, -0.0, np.nan, 0], np.float32)
    for probs in (True, False):
        x, start, count, tokens, q, u, r = drafts(rng, [3] * len(t), 500, probs=probs)
        x[:, 3] = -np.inf
        check(x, start, count, tokens, q, t, u, r)


def test_drafts_that_cannot_be():
    """Tokens outside the vocabulary, drafts without probability, distributions equal to the target's and above it
    everywhere (nothing is left: the token comes from p), the same draft twice."""
    rng = np.random.default_rng(6)
    x, start, count, tokens, q, u, r = drafts(rng, [4] * 30, 100)
    tokens[1::4][:10] = [-1, 100, 1 << 30, -(1 << 31), 99, 0, 101, -5, 100, 7]
    check(x, start, count, tokens, q, None, u, r)
    check(x, start, count, tokens, None, None, u, r)
    q[np.arange(len(q) - 1), np.clip(tokens[1:], 0, 99)] = 0
    check(x, start, count, tokens, q, None, u, r)
    q[:] = 2.0
    got = check(x, start, count, tokens, q, None, u, r)
    assert np.all(got[2][start + got[0]] >= 0)
    p = np.exp(x.astype(np.float64))
    q = (p / p.sum(-1, keepdims=True)).astype(np.float32)
    check(x, start, count, tokens, q, None, np.minimum(u, np.float32(0.999)), r)


def test_equal_logits():
    """Greedy ties go to the lower id, draws among equal tokens follow the random number."""
    x = np.zeros((6, 1000), np.float32)
    x[:, 400:500] = 3.0
    x[3, 400:500] = -0.0
    tokens = np.array([0, 400, 401, 0, 0, 399], np.int32)
    r = np.array([0.5, 0.25], np.float32)
    got = check(x, [0, 3], [3, 3], tokens, None, np.zeros(2, np.float32), np.zeros(6, np.float32), r)
    assert got[0].tolist() == [1, 1] and got[2].tolist() == [400, 400, -1, 0, 400, -1]
    check(x, [0, 3], [3, 3], tokens, None, None, np.zeros(6, np.float32), r)


def test_a_row_may_be_drawn_alone():
    """Requests of one row draw a token each, distributed as p."""
    rng = np.random.default_rng(7)
    n = 4000
    x = np.log(np.array([[0.5, 0.2, 0.2, 0.1]])).astype(np.float32).repeat(n, 0)
    r = ((np.arange(n) + 0.5) / n).astype(np.float32)
    got = check(x, np.arange(n), np.ones(n, int), np.zeros(n, int), None, None, np.zeros(n), r)
    # evenly spaced numbers: shares to one of n, and the logits' rounding to 2^-24
    np.testing.assert_allclose(np.bincount(got[2]) / n, [0.5, 0.2, 0.2, 0.1], atol=1.5 / n)


def test_repeats_and_graphs():
    """The same call twice, and captured and replayed between other work, gives the same numbers."""
    rng = np.random.default_rng(8)
    x, start, count, tokens, q, u, r = drafts(rng, [5, 1, 3, 5], 20000)
    want = check(x, start, count, tokens, q, None, u, r)
    rows, vocab = x.shape
    nb = rehip.draft_verify_work_bytes(rows, 4, vocab)
    d = [B.from_array(x), i32(start), i32(count), i32(tokens), B.from_array(q), B.from_array(u), B.from_array(r)]
    o = [i32(np.full(4, -5)), i32(np.full(4, -5)), i32(np.full(rows, -5))]
    work, stream = B(nb), hip.Stream()
    call = lambda: rehip.draft_verify_dev(d[0], vocab, rows, vocab, 4, d[1], d[2], d[3], d[4], vocab, None, d[5], d[6], *o,  # noqa: E731
                                          work, nb, stream)
    graph = hip.Graph(stream, call)
    for i in range(3):
        for buf in o:
            buf.upload(np.full(buf.nbytes // 4, -5, np.int32))
        hip.synchronize()
        graph.launch()
        stream.synchronize()
        for buf, w in zip(o, want):
            np.testing.assert_array_equal(get(buf, len(w)), w)
        check(x, start, count, tokens, None, None, u, r)
    graph.destroy()
    stream.destroy()
