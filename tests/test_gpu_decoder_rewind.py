"""DeviceDecoder taken back to its first tokens: `seq_len` is all that a caller sets, on both caches."""
import numpy as np
import pytest

from rehip import qwen

pytestmark = pytest.mark.gpu

GEOM = qwen.Geometry(d_model=256, n_heads=4, n_kv_heads=2, d_ff=512, rope_freq_base=1e4, rms_eps=1e-5)


@pytest.fixture(scope="module")
def tiny():
    return qwen.synth_model(7, GEOM, n_layers=3, n_vocab=1000)


def decoder(mb, kv_cache, use_graph=True):
    return qwen.DeviceDecoder(mb, max_seq=400, prefill_rows=200, kv_cache=kv_cache, use_graph=use_graph)


def token(dd, t):
    dd.tok.upload(np.array([t], np.int32))


@pytest.mark.parametrize("use_graph", [True, False])
@pytest.mark.parametrize("kv_cache", ["f32", "int8"])
def test_another_prompt_after_setting_back(tiny, kv_cache, use_graph):
    """A second conversation, and one that keeps its first 64 tokens, give a new decoder's tokens and logits."""
    rng = np.random.default_rng(50)
    first, other, rest = (rng.integers(0, 1000, n) for n in (100, 70, 41))
    dd = decoder(tiny, kv_cache, use_graph)
    dd.generate(first, 30)
    dd.seq_len = 0
    tokens = [dd.generate(other, 25)]
    logits = [dd.logits()]
    dd.seq_len = 0
    dd.prefill(first[:64])
    dd.generate(other, 3)
    dd.seq_len = 64
    tokens.append(dd.generate(rest, 20))
    logits.append(dd.logits())
    dd.close()
    for kept, prompt, n in ((None, other, 25), (first[:64], rest, 20)):
        new = decoder(tiny, kv_cache, use_graph)
        if kept is not None:
            new.prefill(kept)
        assert new.generate(prompt, n) == tokens.pop(0)
        np.testing.assert_array_equal(new.logits(), logits.pop(0))
        new.close()


@pytest.mark.parametrize("use_graph", [True, False])
@pytest.mark.parametrize("kv_cache", ["f32", "int8"])
def test_steps_after_setting_back(tiny, kv_cache, use_graph):
    """Steps and replays from a position that was passed before repeat what they gave there."""
    prompt = np.random.default_rng(51).integers(0, 1000, 64)
    dd = decoder(tiny, kv_cache, use_graph)
    t0 = dd.prefill(prompt)
    want = [dd.step() for _ in range(70)]
    logits = dd.logits()
    dd.seq_len = 64
    token(dd, t0)
    assert [dd.step() for _ in range(70)] == want
    np.testing.assert_array_equal(dd.logits(), logits)
    dd.seq_len = 64
    token(dd, t0)
    dd.replay(70)
    assert dd.history(65, 70) == want and dd.seq_len == 134
    np.testing.assert_array_equal(dd.logits(), logits)
    dd.seq_len = 0                                          # (a decoder also steps from nothing)
    token(dd, 5)
    got = [dd.step() for _ in range(3)]
    dd.close()
    new = decoder(tiny, kv_cache, use_graph)
    token(new, 5)
    assert [new.step() for _ in range(3)] == got
    new.close()


def test_positions_that_the_sequence_does_not_have(tiny):
    for kv_cache, bad in (("f32", (-1, 401)), ("int8", (-1, 21, 400))):
        dd = decoder(tiny, kv_cache)
        dd.prefill(np.arange(20))
        for n in bad:
            with pytest.raises(ValueError):
                dd.seq_len = n
        assert dd.seq_len == 20
        dd.seq_len = 20
        dd.close()


@pytest.mark.parametrize("kv_cache", ["f32", "int8"])
def test_calls_that_fail_leave_the_sequence(tiny, kv_cache, monkeypatch):
    """A prefill and a scoring that raise on their way (no memory, say): the next step goes on where the sequence was."""
    import rehip
    prompt = np.random.default_rng(52).integers(0, 1000, 64)
    dd = decoder(tiny, kv_cache)
    t0 = dd.prefill(prompt)
    want = [dd.step() for _ in range(5)]
    logits = dd.logits()
    for call, name in ((dd.prefill, "add_dev"), (dd.score, "logprobs_dev")):
        dd.seq_len = 64
        with monkeypatch.context() as m:
            def fail(*a, **k):
                raise RuntimeError("no memory")
            m.setattr(rehip, name, fail)
            with pytest.raises(RuntimeError):
                call(prompt[:30])
        assert dd.seq_len == 64
        token(dd, t0)
        assert [dd.step() for _ in range(5)] == want
        np.testing.assert_array_equal(dd.logits(), logits)
    dd.close()


def test_prefills_past_what_a_plan_takes():
    """The plan of int8 pages takes up to 262144 new tokens of a request: a longer prefill is refused, not run on
    rows without a place, and the decoder goes on as if it had not been asked."""
    g = qwen.Geometry(d_model=32, n_heads=1, n_kv_heads=1, d_ff=32, rope_freq_base=1e4, rms_eps=1e-5)
    dd = qwen.DeviceDecoder(qwen.synth_model(9, g, n_layers=1, n_vocab=64), max_seq=(1 << 18) + 100,
                            prefill_rows=(1 << 18) + 1, kv_cache="int8")
    first = dd.prefill([3, 4, 5])
    for call in (dd.prefill, dd.score):
        with pytest.raises(ValueError):
            call(np.zeros((1 << 18) + 1, np.int32))
    dd.seq_len = 0
    assert dd.prefill([3, 4, 5]) == first
    logits = []
    prompt = np.random.default_rng(53).integers(0, 64, 1 << 18)
    for n in (1 << 16, 1 << 18):                            # the longest prefill is what its parts are
        dd.seq_len = 0
        for i in range(0, 1 << 18, n):
            dd.prefill(prompt[i:i + n])
        logits.append(dd.logits())
    assert qwen.logit_profile_check(*logits)["ok"]
    dd.close()


def test_score_of_a_prompt_with_a_batch_axis(tiny):
    """prefill() takes prompts of any shape; scoring one gives a target to every row."""
    prompt = np.random.default_rng(54).integers(0, 1000, 30)
    dd = decoder(tiny, "f32")
    want = dd.score(prompt, 3)
    for shaped in (prompt[None], prompt.reshape(5, 6), prompt.tolist()):
        dd.seq_len = 0
        got = dd.score(shaped, 3)
        assert got["next"] == want["next"]
        for k in ("logprob", "entropy", "ids", "top"):
            np.testing.assert_array_equal(got[k], want[k])
    dd.close()
