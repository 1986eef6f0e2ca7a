"""Page moves whose pages end at, before and behind the end of a workgroup's
segment (4 KB of a copy, 8 KB of a compaction), and refusals that move nothing."""

import numpy as np
import pytest
import torch

import microserve_amd as M
from tests.test_gpu_kv_blocks import _check_compact

pytestmark = pytest.mark.gpu

DEV = "cuda"
# around one, two and several segments of either kind
PAGES = [16, 2048, 4080, 4096, 4112, 8176, 8192, 8208, 12272, 12288, 12304, 16400, 24560, 24592,
         50000]


def _pool(gen, planes, pages, size):
    return torch.randint(0, 256, (planes, pages, size), generator=gen, dtype=torch.uint8).to(DEV)


@pytest.mark.parametrize("size", PAGES)
def test_copies_of_pages_that_end_inside_a_segment(size):
    pool = _pool(torch.Generator().manual_seed(size), 3, 9, size)
    want = pool.clone()
    want[:, [8, 0, 3]] = want[:, [1, 2, 1]]
    M.copy_kv_blocks(pool, [1, 2, 1], [8, 0, 3], block_dim=1)
    assert torch.equal(pool, want)


@pytest.mark.parametrize("size", PAGES)
def test_compaction_of_pages_that_end_inside_a_segment(size):
    pool = _pool(torch.Generator().manual_seed(size + 1), 3, 40, size)
    _check_compact([pool], np.array([[39, 3, -1], [17, 20, 22], [39, 38, 1]], np.int32), None, 1)


def test_compaction_of_pools_of_unlike_pages():
    """One launch's segments of all the sizes, and two launches' worth."""
    gen = torch.Generator().manual_seed(3)
    tables = np.array([[29, 3, -1], [17, 20, 22], [28, 5, 29]], np.int32)
    for sizes in (PAGES[2:10], PAGES):
        _check_compact([_pool(gen, 1 + i % 3, 30, n) for i, n in enumerate(sizes)], tables, 29, 1)


@pytest.mark.parametrize("at", [0, 7, 8, 16])
def test_a_refused_tensor_leaves_the_others_as_they_were(at):
    gen = torch.Generator().manual_seed(4)
    pools = [_pool(gen, 2, 12, 4096 + 16 * i) for i in range(17)]
    pools[at] = _pool(gen, 2, 12, 24)
    before = [p.clone() for p in pools]
    tables = torch.tensor([[11, 2, 9]], dtype=torch.int32, device=DEV)
    with pytest.raises(RuntimeError, match="not supported"):
        M.copy_kv_blocks(pools, [1, 3], [0, 2], block_dim=1)
    with pytest.raises(RuntimeError, match="not supported"):
        M.compact_kv_blocks(pools, tables, block_dim=1)
    for p, b in zip(pools, before):
        assert torch.equal(p, b)
