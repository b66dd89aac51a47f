"""DeviceDecoder on int8 pages, and its scoring of a prompt."""
import numpy as np
import pytest

from rehip import qwen

pytestmark = pytest.mark.gpu

GEOM = qwen.Geometry(d_model=256, n_heads=4, n_kv_heads=2, d_ff=512, rope_freq_base=1e4, rms_eps=1e-5)


@pytest.fixture(scope="module")
def tiny():
    return qwen.synth_model(7, GEOM, n_layers=3, n_vocab=1000)


def logits_of(mb, prompt, steps, **k):
    dd = qwen.DeviceDecoder(mb, max_seq=400, prefill_rows=200, **k)
    toks, lg = [dd.prefill(prompt)], [dd.logits()]
    for _ in range(steps):
        toks.append(dd.step())
        lg.append(dd.logits())
    dd.close()
    return toks, np.stack(lg)


def test_int8_pages_pass_the_logit_profile_gate(tiny):
    """Prompt and steps over page borders against the f32 caches, token by token as the f32 decoder chose them: the
    gate that the bf16 paths pass (gaps of the five best within 0.75 nats, the argmax where it is decisive)."""
    prompt = np.random.default_rng(1).integers(0, 1000, 150)
    want, lw = logits_of(tiny, prompt, 60)
    dd = qwen.DeviceDecoder(tiny, max_seq=400, prefill_rows=200, kv_cache="int8")
    dd.prefill(prompt)
    for i, t in enumerate(want[:-1]):
        gate = qwen.logit_profile_check(lw[i], dd.logits())
        assert gate["ok"], (i, gate)
        dd.tok.upload(np.array([t], np.int32))
        dd.step()
    dd.close()


def test_int8_graph_steps_equal_eager_ones(tiny):
    prompt = np.random.default_rng(2).integers(0, 1000, 61)
    a, la = logits_of(tiny, prompt, 80, kv_cache="int8", use_graph=True)
    b, lb = logits_of(tiny, prompt, 80, kv_cache="int8", use_graph=False)
    assert a == b
    np.testing.assert_array_equal(la, lb)


def test_int8_new_conversations_and_replays(tiny):
    """A second conversation on the same decoder, several prompts in one, and steps without synchronisation give
    what a new decoder gives."""
    prompt = np.random.default_rng(3).integers(0, 1000, 100)
    dd = qwen.DeviceDecoder(tiny, max_seq=400, prefill_rows=200, kv_cache="int8")
    first = dd.generate(prompt, 30)
    dd.seq_len = 0
    dd.pos.zero()
    assert dd.generate(prompt, 30) == first
    dd.seq_len = 0
    dd.pos.zero()
    dd.prefill(prompt[:40])
    dd.prefill(prompt[40:])
    chunked = dd.logits()
    dd.close()
    whole = logits_of(tiny, prompt, 0, kv_cache="int8")[1][0]
    # the first 40 rows' page is filled in two parts: its codes are rounded to another scale in between
    assert qwen.logit_profile_check(whole, chunked)["ok"]


def test_int8_a_sequence_set_back(tiny):
    """Tokens behind a page boundary taken back: what follows is as if they had never been there."""
    rng = np.random.default_rng(5)
    prompt, other = rng.integers(0, 1000, 100), rng.integers(0, 1000, 150)
    got = []
    for detour in (False, True):
        dd = qwen.DeviceDecoder(tiny, max_seq=400, prefill_rows=200, kv_cache="int8")
        dd.prefill(prompt[:64])
        if detour:
            dd.prefill(other)
            dd.step()
            dd.seq_len = 64
            dd.pos.upload(np.array([64], np.int32))
        tokens = [dd.prefill(prompt[64:])] + [dd.step() for _ in range(8)]
        got.append((tokens, dd.logits()))
        dd.close()
    assert got[0][0] == got[1][0]
    np.testing.assert_array_equal(got[0][1], got[1][1])


@pytest.mark.parametrize("kv_cache", ["f32", "int8"])
def test_score(tiny, kv_cache):
    """Each row's numbers are those of the logits that prefilling up to it gives; the sequence goes on as after
    prefill."""
    prompt = np.random.default_rng(4).integers(0, 1000, 133)
    dd = qwen.DeviceDecoder(tiny, max_seq=400, prefill_rows=200, kv_cache=kv_cache)
    got = dd.score(prompt, 5)
    assert got["next"] == int(np.argmax(dd.logits()))
    after = [dd.step() for _ in range(5)]
    plain = qwen.DeviceDecoder(tiny, max_seq=400, prefill_rows=200, kv_cache=kv_cache)
    assert plain.prefill(prompt) == got["next"] and [plain.step() for _ in range(5)] == after
    for r in (0, 1, 63, 64, 100, 132):
        plain.seq_len = 0
        plain.pos.zero()
        plain.prefill(prompt[:r + 1])
        x = plain.logits().astype(np.float64)
        lp = x - x.max() - np.log(np.exp(x - x.max()).sum())
        # the row's logits by another GEMM (and, on int8 pages, scales of the prompt's later rows): the gate's
        # tolerance there, f32 sums' here
        tol = 0.75 if kv_cache == "int8" else 2e-3
        assert abs(got["logprob"][r] - (lp[prompt[r + 1]] if r < 132 else 0)) <= tol
        assert abs(got["entropy"][r] + (np.exp(lp) * lp).sum()) <= tol
        assert np.all(np.abs(got["top"][r] - lp[got["ids"][r]]) <= tol)
        assert np.all(np.diff(got["top"][r]) <= 0)
    plain.close()
    only = dd.score(prompt[:7])
    assert set(only) == {"logprob", "entropy", "next"} and only["logprob"][6] == 0
    for bad in (-1, 65):
        with pytest.raises(ValueError):
            dd.score(prompt[:7], bad)
    dd.close()


def test_unknown_caches_are_refused(tiny):
    with pytest.raises(ValueError):
        qwen.DeviceDecoder(tiny, max_seq=64, kv_cache="int4")
    odd = qwen.synth_model(7, qwen.Geometry(d_model=192, n_heads=4, n_kv_heads=2, d_ff=256, rope_freq_base=1e4,
                                            rms_eps=1e-5), n_layers=1, n_vocab=64)
    with pytest.raises(ValueError):
        qwen.DeviceDecoder(odd, max_seq=64, kv_cache="int8")
