"""The entry points for long conversations and drafted tokens without a GPU: refusals come before any launch; the plain
restatements that the GPU is held to agree with what they restate."""
import ctypes
import math

import numpy as np
import pytest

import keep_ref as ref
import rehip
import serving_ref

A, B = 1 << 20, 1 << 21          # addresses that are never read: every call here is refused first
ARG, SIZE = rehip.RE_ERR_ARG, rehip.RE_ERR_SIZE


def refused(code, fn, *a, **k):
    with pytest.raises(rehip.RehipError) as e:
        fn(*a, **k)
    assert e.value.code == code, e.value
    return e.value.message


def nulls(*names):
    return [(ARG, {k: None}) for k in names]


BATCH = dict(rows=8, requests=2, row_start=A, row_count=A, kv_len=A, table=A, table_ld=4, page=64, n_pages=9, kcodes=A,
             kscale=A, n_kv_heads=2, head_dim=64, q=A, ldq=512, max_rows=4, max_len=256, n_heads=8, scale=0.125,
             window=100, sinks=4, lse=A)
ATTN = dict(BATCH, vcodes=A, vscale=A, ctx=A, work=A, work_bytes=1 << 40)
MASS = dict(BATCH, mass=A)
BAD = nulls("row_start", "row_count", "kv_len", "table", "kcodes", "kscale", "q") + [
    (ARG, {"kcodes": A + 8}), (ARG, {"q": A + 4}), (ARG, {"scale": math.nan}), (ARG, {"scale": math.inf}),
    *[(SIZE, c) for c in ({"page": 0}, {"page": 48}, {"page": 288}, {"head_dim": 80}, {"head_dim": 288}, {"head_dim": 0},
                          {"n_kv_heads": 0}, {"n_kv_heads": 1025}, {"table_ld": 0}, {"table_ld": 1 << 25}, {"n_pages": 0},
                          {"n_pages": 1 << 25}, {"rows": (1 << 22) + 1}, {"requests": 65537}, {"n_heads": 0},
                          {"n_heads": 7}, {"n_heads": 8194}, {"ldq": 508}, {"ldq": 514}, {"max_rows": 0},
                          {"sinks": 1025})]]


@pytest.mark.parametrize("code,change", BAD + nulls("vcodes", "vscale", "ctx") + [
    (ARG, {"ctx": A + 8}), (ARG, {"work": A + 4}), (ARG, {"vcodes": A + 1})])
def test_attention_refusals(code, change):
    refused(code, rehip.attention_kv8_sinks_dev, **{**ATTN, **change})


def test_attention_short_workspaces_are_refused():
    a = dict(ATTN, rows=1, max_len=1 << 17)
    need = rehip.attention_kv8_work_bytes(1, 2, 4, 1 << 17, 8, 2, 64)
    assert need > 0
    refused(SIZE, rehip.attention_kv8_sinks_dev, **{**a, "work_bytes": need - 1})
    refused(ARG, rehip.attention_kv8_sinks_dev, **{**a, "work": None, "work_bytes": 0})


@pytest.mark.parametrize("code,change", BAD + nulls("lse", "mass") + [
    (ARG, {"mass": A + 8}), (SIZE, {"requests": 65536, "n_kv_heads": 256, "n_heads": 256, "ldq": 256 * 64})])
def test_mass_refusals(code, change):
    refused(code, rehip.kv8_mass_dev, **{**MASS, **change})


PLAN = dict(requests=4, page=64, limit=200, keep=100, kv_len=A, table=A, table_ld=8, free=A, n_pages=16, n_free=A,
            kv_len_out=A, table_out=B, free_out=A, n_free_out=A, from_len=A, from_table=A, dropped=None, status=A)
POOL = [(SIZE, c) for c in ({"requests": 0}, {"requests": 4097}, {"page": 0}, {"table_ld": 0}, {"table_ld": 1 << 25},
                            {"n_pages": 0}, {"n_pages": 1 << 25}, {"requests": 4096, "table_ld": (1 << 18) + 1})]


@pytest.mark.parametrize("code,change", POOL + nulls(
    "kv_len", "table", "free", "n_free", "kv_len_out", "table_out", "free_out", "n_free_out", "from_len", "from_table",
    "status") + [(SIZE, {"keep": 0}), (SIZE, {"keep": 201}), (SIZE, {"keep": (1 << 30) + 1, "limit": 1 << 31}), (ARG, {"table_out": A}),
                 (SIZE, {"page": 65537})])
def test_evict_plan_refusals(code, change):
    refused(code, rehip.kv_evict_plan_dev, **{**PLAN, **change})


@pytest.mark.parametrize("same", ["kv_len", "kv_len_out"])
def test_evict_plan_keeps_old_lengths_apart(same):
    refused(ARG, rehip.kv_evict_plan_dev, **{**PLAN, "kv_len": A + 64, "kv_len_out": A + 128, same: A})


EVICT = dict(requests=4, from_len=A, from_table=A, table=B, table_ld=8, page=64, n_pages=16, kcodes=A, vcodes=A, kscale=A,
             vscale=A, mass=A, n_kv_heads=2, head_dim=64, keep=100, first=4, recent=50, max_len=300, kept=A)


@pytest.mark.parametrize("code,change", POOL + nulls("from_len", "from_table", "table", "kcodes", "vcodes", "kscale", "vscale",
                                                     "kept") + [
    (ARG, {"table": A}), (ARG, {"mass": None}), (ARG, {"mass": A + 8}), (ARG, {"kcodes": A + 8}), (ARG, {"vcodes": A + 4}),
    *[(SIZE, c) for c in ({"keep": 0}, {"keep": (1 << 30) + 1}, {"first": 101}, {"recent": 97}, {"first": 100, "recent": 1},
                          {"page": 48}, {"page": 288}, {"head_dim": 80}, {"head_dim": 0}, {"n_kv_heads": 0},
                          {"requests": 4096, "n_kv_heads": 1024}, {"first": (1 << 64) - 1, "recent": 2},
                          {"requests": 2048, "n_kv_heads": 1024, "keep": 1 << 16, "table_ld": 1 << 10, "page": 64})]])
def test_evict_refusals(code, change):
    refused(code, rehip.kv8_evict_dev, **{**EVICT, **change})


REWIND = dict(requests=4, page=64, back=A, kv_len=A, table=A, table_ld=8, free=A, n_pages=16, n_free=A, kv_len_out=A,
              n_free_out=A)


@pytest.mark.parametrize("code,change", POOL + [(SIZE, {"page": 65537})] + nulls(
    "back", "kv_len", "table", "free", "n_free", "kv_len_out", "n_free_out"))
def test_rewind_refusals(code, change):
    refused(code, rehip.kv_rewind_dev, **{**REWIND, **change})


VERIFY = dict(logits=A, ld=1000, rows=9, vocab=1000, requests=3, row_start=A, row_count=A, tokens=A, probs=A, ldp=1000,
              temperature=A, accept_u=A, sample_u=A, accepted=A, back=A, out_tokens=A, work=A, work_bytes=1 << 40)


@pytest.mark.parametrize("code,change", nulls("logits", "row_start", "row_count", "tokens", "accept_u", "sample_u", "accepted",
                                              "back", "out_tokens", "work") + [
    (ARG, {"work": A + 8}),
    *[(SIZE, c) for c in ({"vocab": 0}, {"ld": 999}, {"ldp": 999}, {"vocab": (1 << 24) + 1, "ld": 1 << 25, "ldp": 1 << 25},
                          {"rows": (1 << 22) + 1}, {"requests": 65537}, {"rows": 0}, {"ld": (1 << 30) + 1},
                          {"ldp": (1 << 30) + 1}, {"work_bytes": 8})]])
def test_verify_refusals(code, change):
    refused(code, rehip.draft_verify_dev, **{**VERIFY, **change})


POSITIONS = dict(rows=9, row_seq=A, row_pos=A, requests=3, dropped=A, out=A)


@pytest.mark.parametrize("code,change", nulls("row_seq", "row_pos", "dropped", "out") + [
    (SIZE, {"rows": (1 << 22) + 1}), (SIZE, {"requests": 0}), (SIZE, {"requests": 65537})])
def test_positions_refusals(code, change):
    refused(code, rehip.kv_positions_dev, **{**POSITIONS, **change})


def test_no_rows_is_no_work():
    rehip.kv_positions_dev(**{**POSITIONS, "rows": 0})
    rehip.attention_kv8_sinks_dev(**{**ATTN, "rows": 0, "work": None, "work_bytes": 0})
    rehip.kv8_mass_dev(**{**MASS, "rows": 0})
    rehip.draft_verify_dev(**{**VERIFY, "requests": 0, "rows": 0})
    assert rehip.draft_verify_work_bytes(0, 1, 100) == 0 and rehip.draft_verify_work_bytes(1, 0, 100) == 0


class View:
    """What else may stand for an address or a stream."""
    def __init__(self, **k):
        self.__dict__.update(k)


def test_views_and_streams():
    change = {k: View(ptr=A) for k in ("kv_len", "table", "free", "n_free", "back", "kv_len_out")}
    refused(SIZE, rehip.kv_rewind_dev, **{**REWIND, **change, "stream": View(handle=0), "page": 0})
    refused(SIZE, rehip.kv_rewind_dev, **{**REWIND, "page": 0, "stream": 0})
    with pytest.raises(ctypes.ArgumentError):
        rehip.kv_rewind_dev(**{**REWIND, "table": 1.5, "page": 0})


# ---- the plain restatements ----------------------------------------------------------------------
def test_plain_attention_without_sinks_is_the_plain_attention():
    rng = np.random.default_rng(1)
    kc, vc = (rng.integers(-128, 128, (5, 2, 32, 32)).astype(np.int8) for _ in range(2))
    ks, vs = (np.exp(rng.standard_normal((5, 2))).astype(np.float32) / 50 for _ in range(2))
    batch = (np.array([0, 3]), np.array([3, 1]), np.array([40, 70]), np.array([[0, 1, -1], [2, 3, 4]]), 32)
    q = rng.standard_normal((4, 4, 32)).astype(np.float32)
    want, got, lse = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape[:2])
    serving_ref.attention(q, *batch, kc, vc, ks, vs, 0.2, 17, want)
    ref.attention(q, batch, (kc, vc, ks, vs), 0.2, 17, 0, got, lse)
    np.testing.assert_allclose(got, want, rtol=1e-12)
    # the weights of a row's tokens sum to one for each query head
    m = np.zeros((5, 2, 32))
    ref.mass(q, lse, batch, kc, ks, 0.2, 17, 0, m)
    np.testing.assert_allclose(m.sum(), 4 * 4, rtol=1e-12)


def test_plain_verification_draws_from_the_target():
    """Over many random numbers, drafts from q and the token behind are distributed as p (that is what the rule is for)."""
    rng = np.random.default_rng(2)
    n, vocab = 40000, 5
    x = np.log(np.array([0.4, 0.3, 0.2, 0.1, 0.0]) + 1e-300).astype(np.float32)
    q = np.array([0.1, 0.2, 0.3, 0.2, 0.2], np.float32)
    drafts = rng.choice(vocab, n, p=q.astype(np.float64) / q.astype(np.float64).sum())
    out = np.zeros(2 * n, np.int32)
    tokens = np.stack([np.zeros(n, int), drafts], 1).reshape(-1)
    ref.verify(np.tile(x, (2 * n, 1)), 2 * np.arange(n), np.full(n, 2), tokens, np.tile(q, (2 * n, 1)), None,
               rng.random(2 * n), rng.random(n), out)
    share = np.bincount(out[::2], minlength=vocab) / n
    # three standard deviations of a share of 0.4 of 40000: 0.0074
    np.testing.assert_allclose(share, [0.4, 0.3, 0.2, 0.1, 0.0], atol=0.0074)
