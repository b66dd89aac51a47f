"""Log probabilities of long flat rows: the sums of many equal terms do not drift."""
import ctypes as C

import numpy as np
import pytest

import rehip
import serving_ref as ref
from rehip import hip
from test_gpu_serve_ops import EPS, get, i32

pytestmark = pytest.mark.gpu
B = hip.DeviceBuffer


def drift(c, n):
    """4 and n times c added one after the other in f32, off by how much of the sum"""
    z = np.full_like(c, 4)
    for _ in range(n):
        z = z + c
    exact = 4 + n * c.astype(np.float64)
    return np.abs(z - exact) / exact


@pytest.mark.parametrize("rows,vocab", [(1536, 151936), (400, 151936), (1, 1 << 24)])
def test_sums_of_equal_terms(rows, vocab):
    """A row's first 4096 logits hold a 0 for every lane and the others are all alike, at values whose repeated f32 sum
    rounds the same way every time: added one after the other, 2370 of them to a lane, ln Z is off by up to 590 EPS.

    The bound: a term is off by 6 EPS (d, its product with log2 e, exp2), 16 of them summed by 15, the batches' sum with
    its rounding errors kept by 2, the joins of lanes, waves and parts by 16, the logarithm by 2 ulp of ln Z (up to 17: 68 EPS)
    and the last differences by 2 of 18; the entropy has T / Z (up to 1.3 in size, twice the sums' errors) beside it."""
    rng = np.random.default_rng(80)
    c = rng.uniform(0.3, 1, 3000).astype(np.float32)
    worst = c[np.argsort(drift(c, 2370))[-16:]]
    x = np.repeat(np.log(worst.astype(np.float64)).astype(np.float32)[:, None], vocab, 1)[:min(rows, 16)]
    x[:, :4096].reshape(len(x), 4, 1024)[..., :256] = 0     # (four for each lane of each of four waves)
    buf = B(rows * vocab * 4)
    for r in range(0, rows, 16):
        part = np.ascontiguousarray(x[:min(16, rows - r)])
        hip.check(hip.hip().hipMemcpy(C.c_void_p(buf.ptr + 4 * r * vocab), part.ctypes.data, part.nbytes, hip.H2D))
    nb = rehip.logprobs_work_bytes(rows, vocab, 0)
    lp, en, work = B(rows * 4), B(rows * 4), B(max(nb, 16))
    t = np.full(rows, 77, np.int32)
    rehip.logprobs_dev(buf, vocab, rows, vocab, i32(t), 0, lp, en, None, None, work, nb)
    want = ref.logprobs(x, t[:len(x)], 1)
    at = np.arange(rows) % 16
    assert np.abs(get(lp, rows) - want[0][at]).max() <= (6 + 15 + 2 + 16 + 68 + 36) * EPS
    assert np.abs(get(en, rows) - want[1][at]).max() <= (6 + 15 + 2 + 16 + 68 + 36 + 3 * 39) * EPS
