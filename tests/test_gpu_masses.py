"""A step's weights (kv8_mass_dev) against keep_ref.py in 64 bits: calls that attention takes, and what drafted steps leave."""
import numpy as np
import pytest

from test_gpu_attention_sinks import check_mass
from test_gpu_kv8 import make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("max_rows", [1 << 31, 1 << 40, (1 << 64) - 1])
def test_any_bound_of_the_rows(max_rows):
    """max_rows beyond all rows bounds nothing, as in attention."""
    rng = np.random.default_rng(1)
    bt, cache, q = make(rng, [3, 0, 20], [50, 7, 90], 32, 8, 2, 64)
    check_mass(cache, bt, q, 0.125, 30, 4, max_rows=max_rows, max_len=90)
