"""The batched serving entry points without a GPU: refusals come before any launch, the rotary frequencies
follow their formulas."""
import math

import numpy as np
import pytest

import rehip

A, B = 1 << 20, 1 << 21          # addresses that are never read: every call here is refused first


def refused(code, fn, *a, **k):
    with pytest.raises(rehip.RehipError) as e:
        fn(*a, **k)
    assert e.value.code == code, e.value
    return e.value.message


PLAN = dict(requests=4, page=64, new_len=A, kv_len=A, table=A, table_ld=8, free=A, n_pages=16, n_free=A, kv_len_out=A,
            n_free_out=A, row_start=A, row_count=A, row_cap=64, row_seq=A, row_pos=A, row_slot=A, status=A)


@pytest.mark.parametrize("code,change", [
    *[(rehip.RE_ERR_ARG, {k: None}) for k in ("new_len", "kv_len", "table", "free", "n_free", "kv_len_out",
                                              "n_free_out", "row_start", "row_count", "row_seq", "row_pos",
                                              "row_slot", "status")],
    *[(rehip.RE_ERR_SIZE, c) for c in ({"requests": 0}, {"requests": 4097}, {"page": 0}, {"page": 65537},
                                       {"table_ld": 0}, {"table_ld": 1 << 25}, {"n_pages": 0}, {"n_pages": 1 << 25},
                                       {"row_cap": (1 << 22) + 1},
                                       {"requests": 4096, "table_ld": (1 << 18) + 1})]])
def test_plan_refusals(code, change):
    refused(code, rehip.kv_plan_dev, **{**PLAN, **change})


ROPE = dict(x=A, ldx=512, rows=3, heads=4, head_dim=128, rot_dim=64, layout=rehip.ROPE_HALF, freqs=A, mscale=1.0,
            pos=A, out=B, ldo=512)


@pytest.mark.parametrize("code,change", [
    *[(rehip.RE_ERR_ARG, c) for c in ({"x": None}, {"freqs": None}, {"pos": None}, {"out": None}, {"layout": 2},
                                      {"out": A, "ldo": 516})],
    *[(rehip.RE_ERR_SIZE, c) for c in ({"rot_dim": 0}, {"rot_dim": 33}, {"rot_dim": 130}, {"head_dim": 0},
                                       {"head_dim": 257, "ldx": 2048, "ldo": 2048}, {"ldx": 511}, {"ldo": 511},
                                       {"rows": (1 << 22) + 1}, {"heads": 65536, "ldx": 1 << 24, "ldo": 1 << 24})]])
def test_rope_refusals(code, change):
    refused(code, rehip.rope_rows_dev, **{**ROPE, **change})


BATCH = dict(rows=8, requests=2, row_start=A, row_count=A, kv_len=A, table=A, table_ld=4, page=64, n_pages=9, kcodes=A,
             vcodes=A, kscale=A, vscale=A, n_kv_heads=2, head_dim=64)
BAD_BATCH = [
    *[(rehip.RE_ERR_ARG, {k: None}) for k in ("row_start", "row_count", "kv_len", "table", "kcodes", "vcodes", "kscale",
                                              "vscale")],
    (rehip.RE_ERR_ARG, {"kcodes": A + 8}), (rehip.RE_ERR_ARG, {"vcodes": A + 1}),
    *[(rehip.RE_ERR_SIZE, c) for c in ({"page": 0}, {"page": 48}, {"page": 288}, {"head_dim": 80}, {"head_dim": 288},
                                       {"head_dim": 0}, {"n_kv_heads": 0}, {"n_kv_heads": 1025}, {"table_ld": 0},
                                       {"table_ld": 1 << 25}, {"n_pages": 0}, {"n_pages": 1 << 25},
                                       {"rows": (1 << 22) + 1}, {"requests": 65537})]]


@pytest.mark.parametrize("code,change", BAD_BATCH + [
    (rehip.RE_ERR_ARG, {"k": None}), (rehip.RE_ERR_ARG, {"v": None}), (rehip.RE_ERR_ARG, {"k": A + 4}),
    (rehip.RE_ERR_SIZE, {"ldk": 124}), (rehip.RE_ERR_SIZE, {"ldv": 130}),
    (rehip.RE_ERR_SIZE, {"ldv": (1 << 22) + 4})])
def test_append_refusals(code, change):
    refused(code, rehip.kv8_append_dev, **{**BATCH, "k": A, "v": A, "ldk": 128, "ldv": 128, **change})


ATTN = dict(BATCH, q=A, ldq=512, max_rows=4, max_len=256, n_heads=8, scale=0.125, window=0, ctx=A, work=A,
            work_bytes=1 << 40)


@pytest.mark.parametrize("code,change", BAD_BATCH + [
    *[(rehip.RE_ERR_ARG, c) for c in ({"q": None}, {"ctx": None}, {"q": A + 4}, {"ctx": A + 8}, {"work": A + 4},
                                      {"scale": math.nan}, {"scale": math.inf})],
    *[(rehip.RE_ERR_SIZE, c) for c in ({"n_heads": 0}, {"n_heads": 7}, {"n_heads": 8194}, {"ldq": 508}, {"ldq": 514},
                                       {"max_rows": 0},
                                      {"rows": 1 << 22, "max_rows": 1 << 22, "n_heads": 1024, "n_kv_heads": 1024,
                                       "ldq": 65536})]])
def test_attention_refusals(code, change):
    refused(code, rehip.attention_kv8_dev, **{**ATTN, **change})


LOG = dict(logits=A, ld=1000, rows=5, vocab=1000, targets=A, top_k=5, logprob=A, entropy=A, top_ids=A,
           top_logprobs=A, work=A, work_bytes=1 << 40)


@pytest.mark.parametrize("code,change", [
    *[(rehip.RE_ERR_ARG, c) for c in ({"logits": None}, {"targets": None}, {"top_ids": None}, {"top_logprobs": None},
                                      {"work": A + 4})],
    *[(rehip.RE_ERR_SIZE, c) for c in ({"vocab": 0}, {"ld": 999}, {"vocab": (1 << 24) + 1, "ld": 1 << 25},
                                       {"top_k": 65}, {"top_k": 4, "vocab": 3}, {"rows": (1 << 22) + 1})]])
def test_logprobs_refusals(code, change):
    refused(code, rehip.logprobs_dev, **{**LOG, **change})


@pytest.mark.parametrize("fn,args,size", [
    (rehip.attention_kv8_dev, ATTN, lambda a: rehip.attention_kv8_work_bytes(
        a["rows"], a["requests"], a["max_rows"], a["max_len"], a["n_heads"], a["n_kv_heads"], a["head_dim"])),
    (rehip.logprobs_dev, LOG, lambda a: rehip.logprobs_work_bytes(a["rows"], a["vocab"], a["top_k"]))])
def test_short_workspaces_are_refused(fn, args, size):
    a = dict(args, rows=1, max_len=1 << 17) if "max_len" in args else dict(args, vocab=151936, ld=151936)
    need = size(a)
    if need:
        refused(rehip.RE_ERR_SIZE, fn, **{**a, "work_bytes": need - 1})
        refused(rehip.RE_ERR_ARG, fn, **{**a, "work": None, "work_bytes": 0})


def test_no_rows_is_no_work():
    rehip.rope_rows_dev(**{**ROPE, "rows": 0})
    rehip.kv8_append_dev(**{**BATCH, "rows": 0, "k": A, "v": A, "ldk": 128, "ldv": 128})
    rehip.attention_kv8_dev(**{**ATTN, "rows": 0, "work": None, "work_bytes": 0})
    rehip.logprobs_dev(**{**LOG, "rows": 0, "work": None, "work_bytes": 0})
    assert rehip.attention_kv8_work_bytes(0, 1, 1, 100, 8, 2, 64) == 0
    assert rehip.logprobs_work_bytes(0, 1000, 5) == 0


# ---- frequencies -------------------------------------------------------------------------------
def close(got, want):
    # a power, a product and a quotient, each within a few ulp of 2^-53
    np.testing.assert_allclose(got, want, rtol=1e-14, atol=0)


@pytest.mark.parametrize("rot", [2, 6, 64, 128, 256])
@pytest.mark.parametrize("theta", [1e4, 1e6])
def test_frequencies(rot, theta):
    i = np.arange(rot // 2)
    base = theta ** (-2.0 * i / rot)
    f, m = rehip.rope_freqs(theta, rot)
    close(f, base)
    assert m == 1.0
    f, m = rehip.rope_freqs(theta, rot, rehip.ROPE_LINEAR, 4.0)
    close(f, base / 4)
    assert m == 1.0
    if rot > 2:
        f, m = rehip.rope_freqs(theta, rot, rehip.ROPE_NTK, 8.0)
        close(f, (theta * 8.0 ** (rot / (rot - 2))) ** (-2.0 * i / rot))
        assert f[0] == 1.0 and abs(f[-1] * 8 / base[-1] - 1) < 1e-12      # the slowest pair ends up interpolated
    f, m = rehip.rope_freqs(theta, rot, rehip.ROPE_BANDS, 8.0, 8192.0, 1.0, 4.0)
    turns = 8192 * base / (2 * math.pi)
    close(f[turns >= 4], base[turns >= 4])
    close(f[turns <= 1], base[turns <= 1] / 8)
    mid = (turns > 1) & (turns < 4)
    w = (turns[mid] - 1) / 3
    close(f[mid], base[mid] * w + base[mid] / 8 * (1 - w))
    f, m = rehip.rope_freqs(theta, rot, rehip.ROPE_YARN, 16.0, 4096.0)
    assert m == np.float32(0.1 * math.log(16) + 1)
    at = [rot * math.log(4096 / (t * 2 * math.pi)) / (2 * math.log(theta)) for t in (32, 1)]
    low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rot - 1)
    close(f[i <= low], base[i <= low])
    close(f[i >= high], base[i >= high] / 16)
    assert np.all(np.diff(f) < 0)


def test_frequency_refusals():
    for code, a in ((rehip.RE_ERR_SIZE, (1e4, 0)), (rehip.RE_ERR_SIZE, (1e4, 3)), (rehip.RE_ERR_SIZE, (1e4, 258)),
                    (rehip.RE_ERR_ARG, (1.0, 64)), (rehip.RE_ERR_ARG, (math.nan, 64)), (rehip.RE_ERR_ARG, (1e4, 64, 5)),
                    (rehip.RE_ERR_ARG, (1e4, 64, rehip.ROPE_LINEAR, 0.5)),
                    (rehip.RE_ERR_SIZE, (1e4, 2, rehip.ROPE_NTK, 2.0)),
                    (rehip.RE_ERR_ARG, (1e4, 64, rehip.ROPE_YARN, 2.0, 0.0)),
                    (rehip.RE_ERR_ARG, (1e4, 64, rehip.ROPE_BANDS, 2.0, 4096.0, 4.0, 1.0))):
        refused(code, rehip.rope_freqs, *a)
