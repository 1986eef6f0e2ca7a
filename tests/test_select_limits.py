"""The largest calls that the choice of tokens takes."""

import pytest

from microserve_amd import _lib


@pytest.mark.parametrize("batch,heads", [(65535, 65535), (65535, 65), (1024, 4096)])
def test_more_pairs_than_a_grid_holds_are_refused(batch, heads):
    p = 1 << 20  # never read
    assert _lib.load().mskv_select_kv_tokens(p, p, p, None, 0, 0, 4, p, p, batch, heads, 32, 8, 4,
                                             None) == -2
