"""Verified drafts without a GPU: what is refused and asked for before any launch."""
import pytest

import rehip
from test_keep_host import ARG, VERIFY, A, refused


@pytest.mark.parametrize("shift", [0, 4, -4, 4 * 8, -4 * 8])
def test_tokens_do_not_come_out_over_the_drafted_ones(shift):
    """A request's threads write rows that others still read (9 rows: places 8 apart still share one)."""
    assert "apart" in refused(ARG, rehip.draft_verify_dev, **{**VERIFY, "out_tokens": A + shift})
