"""Verified drafts at the edges of their buffers, against keep_ref.py in 64 bits."""
import numpy as np
import pytest

import keep_ref as ref
import rehip
from rehip import hip
from test_gpu_draft_verify import drafts, get
from test_gpu_kv8 import i32

pytestmark = pytest.mark.gpu
B = hip.DeviceBuffer


def f32(a):
    return B.from_array(np.ascontiguousarray(a, np.float32))


@pytest.mark.parametrize("vocab,count", [(2048, [2] * 120 + [17]), (8192, [5] * 13), (8192, [65])])
def test_buffers_that_end_with_the_last_draft(vocab, count):
    """The last row of all has no draft, so neither probabilities nor a random number: 2 MiB of probabilities end before it."""
    rng = np.random.default_rng(vocab + len(count))
    x, start, count, tokens, q, u, r = drafts(rng, count, vocab)
    rows, n = len(x), len(count)
    assert (rows - 1) * vocab * 4 == 1 << 21
    out = np.full(rows, -5, np.int32)
    acc, back = ref.verify(x, start, count, tokens, q, None, u, r, out)
    nb = rehip.draft_verify_work_bytes(rows, n, vocab)
    got = [i32(np.full(n, -5)), i32(np.full(n, -5)), i32(np.full(rows, -5))]
    rehip.draft_verify_dev(f32(x), vocab, rows, vocab, n, i32(start), i32(count), i32(tokens), f32(q[:-1]), vocab, None, f32(u[:-1]),
                           f32(r), *got, B(nb), nb)
    for g, w in zip(got, (acc, back, out)):
        np.testing.assert_array_equal(get(g, len(w)), w)


def test_a_workspace_for_the_largest_step_serves_smaller_ones():
    """Sized once for 1025 rows, which are not cut into parts; fewer rows are cut into two and more."""
    rng, vocab, n = np.random.default_rng(11), 9000, 41
    nb = rehip.draft_verify_work_bytes(1025, n, vocab)
    work = B(nb)
    for per in (25, 12, 6, 1):
        x, start, count, tokens, q, u, r = drafts(rng, [per] * n, vocab, probs=False)
        out = np.full(len(x), -5, np.int32)
        acc, back = ref.verify(x, start, count, tokens, None, None, u, r, out)
        got = [i32(np.full(n, -5)), i32(np.full(n, -5)), i32(np.full(len(x), -5))]
        rehip.draft_verify_dev(f32(x), vocab, len(x), vocab, n, i32(start), i32(count), i32(tokens), None, 0, None, f32(u), f32(r), *got,
                               work, nb)
        for g, w in zip(got, (acc, back, out)):
            np.testing.assert_array_equal(get(g, len(w)), w)


def test_calls_back_to_back_see_their_own_sums():
    """Many calls in one workspace with nothing waited for between them, alternating inputs: a request's last workgroup takes
    the sums of this call, not those that the call before left in the same places."""
    vocab, count = 40000, [4, 1, 3, 5, 2]
    n, rows = len(count), sum(count)
    nb = rehip.draft_verify_work_bytes(rows, n, vocab)
    work, sets = B(nb), []
    for seed in (21, 22):
        rng = np.random.default_rng(seed)
        x, start, count, tokens, q, u, r = drafts(rng, count, vocab, sharp=-20, likely=0.3)
        out = np.full(rows, -5, np.int32)
        want = (*ref.verify(x, start, count, tokens, q, None, u, r, out), out)
        sets.append(((f32(x), i32(start), i32(count), i32(tokens), f32(q), f32(u), f32(r)), want))
    got = [[i32(np.full(n, -5)), i32(np.full(n, -5)), i32(np.full(rows, -5))] for _ in range(60)]
    hip.synchronize()
    for i, o in enumerate(got):
        x, start, count, tokens, q, u, r = sets[i % 2][0]
        rehip.draft_verify_dev(x, vocab, rows, vocab, n, start, count, tokens, q, vocab, None, u, r, *o, work, nb)
    for i, o in enumerate(got):
        for g, w in zip(o, sets[i % 2][1]):
            np.testing.assert_array_equal(get(g, len(w)), w)
