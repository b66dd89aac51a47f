"""Verified drafts without a GPU: what is refused and asked for before any launch."""
import pytest

import rehip
from test_keep_host import ARG, VERIFY, A, refused


@pytest.mark.parametrize("shift", [0, 4, -4, 4 * 8, -4 * 8])
def test_tokens_do_not_come_out_over_the_drafted_ones(shift):
    """A request's threads write rows that others still read (9 rows: places 8 apart still share one)."""
    assert "apart" in refused(ARG, rehip.draft_verify_dev, **{**VERIFY, "out_tokens": A + shift})


def test_the_largest_step_sizes_the_workspace():
    """Sizes never fall as rows, requests or the vocabulary grow."""
    size = rehip.draft_verify_work_bytes
    rows = sorted({*range(1, 70), *(1024 // k + d for k in range(1, 65) for d in (-1, 0, 1)), 1023, 1024, 1025, 4000, 1 << 22} - {0})
    vocabs = [1, 1000, 2048, 2049, 4096, 4097, 32000, 151936, 1 << 20, 1 << 24]
    for vocab in vocabs:
        for requests in (1, 2, 64, 65536):
            sizes = [size(r, requests, vocab) for r in rows]
            assert sizes == sorted(sizes) and sizes[0] > 0
    for r in rows:
        assert [size(r, 64, v) for v in vocabs] == sorted(size(r, 64, v) for v in vocabs)
        assert [size(r, n, 32000) for n in range(1, 70)] == sorted(size(r, n, 32000) for n in range(1, 70))
