"""The largest calls that the choice of tokens takes."""

import pytest
import torch

import microserve_amd as M
from microserve_amd import _lib


@pytest.mark.parametrize("batch,heads", [(65535, 65535), (65535, 65), (1024, 4096)])
def test_more_pairs_than_a_grid_holds_are_refused(batch, heads):
    p = 1 << 20  # never read
    assert _lib.load().mskv_select_kv_tokens(p, p, p, None, 0, 0, 4, p, p, batch, heads, 32, 8, 4,
                                             None) == -2


@pytest.mark.gpu
@pytest.mark.parametrize("budget", [2 ** 31 - 1, 2 ** 31 - 500])
def test_the_largest_budgets(budget):
    """kept of 8 GiB: the last places' numbers and kThreads pass 2^31."""
    weights = torch.zeros(4, 1, 128, device="cuda")
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    kept, n = M.select_kv_tokens(weights, ints(300), ints(3, 1, 0)[None], budget)
    torch.cuda.synchronize()
    assert kept.shape == (1, 1, budget) and int(n) == 300
    flat = kept.view(-1)
    assert torch.equal(flat[:300], torch.arange(300, dtype=torch.int32, device="cuda"))
    for part in flat[300:].split(1 << 28):
        assert int(part.max()) == int(part.min()) == -1
