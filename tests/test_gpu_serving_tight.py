"""Rows that looser bounds elsewhere let pass: scores past 2^20 in wide tiles, the scoring of a prompt's last row on int8
pages."""
import numpy as np
import pytest

import serving_ref as ref
from rehip import qwen
from test_gpu_kv8 import attend, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv_heads,hd,page", [(256, 64, 32, 32), (256, 64, 160, 32)])     # 64 and 32 vectors a tile
@pytest.mark.parametrize("window", [0, 70])
def test_huge_scores_in_wide_tiles(heads, kv_heads, hd, page, window):
    """Where the best score is far above the others, measured by what an f32 score may be off by, the output is that key's
    value; vectors of ordinary scores beside them keep their bound."""
    rng = np.random.default_rng(hd + window)
    bt, cache, q = make(rng, [200, 63], [230, 64], page, heads, kv_heads, hd)
    size = np.ones((bt.rows, 1, 1), np.float32)
    size[40:50], size[90:100, 0], size[230] = 1e20, 3e6, 1e9      # (a score of about 1 times this)
    q *= size
    q[140, ::2] *= np.float32(1e12)                         # every other head of a row
    scale = hd ** -0.5
    want = np.full(q.shape, 7.25)
    tol = ref.attention(q, *bt.plain(), cache.k, cache.v, cache.ks, cache.vs, scale, window, want)
    got = attend(cache, bt, q, scale, window)
    huge = np.abs(q).max(-1) > 1e5
    assert np.all(np.abs(got - want)[~huge] <= tol[~huge][:, None])
    checked = 0
    for r, h in np.argwhere(huge):
        b = int(r >= bt.start[1])
        p = int(bt.len[b] - bt.count[b] + r - bt.start[b])
        j = np.arange(max(0, p - window + 1) if window else 0, p + 1)
        pid, kv = bt.table[b, j // page], h * kv_heads // heads
        k = cache.k[pid, kv, j % page].astype(np.float64) * cache.ks[pid, kv].astype(np.float64)[:, None]
        x = q[r, h].astype(np.float64)
        s = np.sort(k @ x * scale)
        delta = (hd + 16) * 2.0 ** -24 * scale * (np.abs(k) @ np.abs(x)).max()
        if len(s) > 1 and s[-1] - s[-2] < 2 * delta + 40:   # (the others' weight is then below e^-40)
            continue
        checked += 1
        # p in two f16 parts (4 half steps of 2^-24), two sums, the page's scale, the join, 1 / sum and its product
        assert np.all(np.abs(got[r, h] - want[r, h]) <= 16 * 2.0 ** -24 * np.abs(want[r, h]).max()), (r, h)
    assert checked >= 0.8 * np.count_nonzero(huge)


@pytest.mark.parametrize("mode", ["f32", "int8"])
def test_score_of_the_last_row(mode):
    """score() says of its last row what the logits of the same call say. They come from another product of the same
    hidden row: f32 on split operands, within 2^-15 sum |w x| (2^-16 of the parts, 256 sums), here about 5e-4, and twice
    that in a log probability."""
    g = qwen.Geometry(d_model=256, n_heads=4, n_kv_heads=2, d_ff=512, rope_freq_base=1e4, rms_eps=1e-5)
    dd = qwen.DeviceDecoder(qwen.synth_model(7, g, n_layers=3, n_vocab=1000), max_seq=400, prefill_rows=200, kv_cache=mode)
    prompt = np.random.default_rng(70).integers(0, 1000, 200)
    for n in (1, 2, 63, 64, 65, 128, 133, 200):
        dd.seq_len = 0
        got = dd.score(prompt[:n], 64)
        x = dd.logits().astype(np.float64)
        lp = x - x.max() - np.log(np.exp(x - x.max()).sum())
        assert got["next"] == np.argmax(x) and got["logprob"][-1] == 0
        assert abs(got["entropy"][-1] + (np.exp(lp) * lp).sum()) <= 2e-3
        assert np.all(np.abs(got["top"][-1] - lp[got["ids"][-1]]) <= 2e-3)
        assert np.all(np.diff(got["top"][-1]) <= 0) and len(set(got["ids"][-1])) == 64
        assert lp[got["ids"][-1]].min() >= np.sort(lp)[-64] - 4e-3
        if n > 1:                                           # the row before says of the last token: by entropy alone
            assert got["entropy"][-2] <= np.log(1000) + 2e-3 and got["logprob"][-2] < 0
    dd.close()


def test_int8_pages_of_a_decoder_with_unquantized_weights():
    """The bias of a step goes into the q|k|v product: of dense weights that is another kernel. Prompt and steps against
    the f32 caches, by the gate that the bf16 paths pass."""
    from test_gpu_layer import TINY, dense_model
    mb = dense_model(11, TINY, n_layers=3, n_vocab=1000)
    prompt = np.random.default_rng(71).integers(0, 1000, 100)
    a, b = (qwen.DeviceDecoder(mb, max_seq=200, prefill_rows=100, kv_cache=c) for c in ("f32", "int8"))
    t = a.prefill(prompt)
    b.prefill(prompt)
    for i in range(40):
        gate = qwen.logit_profile_check(a.logits(), b.logits())
        assert gate["ok"], (i, gate)
        b.tok.upload(np.array([t], np.int32))
        t = a.step()
        b.step()
    a.close()
    b.close()
