"""The decoder's drafted generation beside its plain one."""
import dataclasses

import numpy as np
import pytest

from rehip import qwen

pytestmark = pytest.mark.gpu
GEOM = qwen.Geometry(d_model=256, n_heads=4, n_kv_heads=2, d_ff=512, rope_freq_base=1e4, rms_eps=1e-5)


@pytest.mark.parametrize("kv_cache", ["f32", "int8"])
def test_generation_without_drafts_is_plain_generation(kv_cache):
    """A model whose every token has a twin of the same logit: single steps take the higher of the two, verified ones the lower.
    Where nothing is drafted (none asked for, or no two tokens that come again) tokens and logits are `generate`'s, bit for bit."""
    mb = qwen.synth_model(9, GEOM, n_layers=2, n_vocab=1000)
    half = np.asarray(mb.output).reshape(2, -1)[0]
    mb = dataclasses.replace(mb, output=np.concatenate([half, half]))
    prompt = np.random.default_rng(2).integers(0, 1000, 40)

    def run(how):
        dd = qwen.DeviceDecoder(mb, max_seq=100, prefill_rows=64, kv_cache=kv_cache)
        got = how(dd), dd.logits(), dd.seq_len
        dd.close()
        return got
    want = run(lambda dd: dd.generate(prompt, 25))
    assert min(want[0]) >= 500
    for how in (lambda dd: dd.generate_drafted(prompt, 25, most=0), lambda dd: dd.generate_drafted(prompt, 25, ngram=40)):
        got = run(how)
        assert got[0] == want[0] and got[2] == want[2]
        np.testing.assert_array_equal(got[1], want[1])
