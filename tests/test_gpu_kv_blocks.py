"""Copies and compaction of a pool's pages against torch indexing and a plain
restatement of the plan."""

import numpy as np
import pytest
import torch

import microserve_amd as M

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _runner_pool(gen, layers, pages, block, heads):
    """The runner's caches and scales, [2, L, NB, ...]."""
    kv = torch.randint(0, 256, (2, layers, pages, block, heads, 128), generator=gen,
                       dtype=torch.uint8).to(DEV).view(torch.float8_e4m3fn)
    sc = torch.rand(2, layers, pages, block, heads, generator=gen).to(DEV)
    return kv, sc


def _bytes(t):
    return t.view(torch.uint8) if t.element_size() == 1 else t.view(torch.int32)


@pytest.mark.parametrize("layers,pages,block,heads,pairs", [
    (1, 2, 256, 1, 1), (3, 9, 128, 5, 4), (2, 40, 256, 8, 20), (1, 700, 32, 1, 300)])
def test_copies_in_every_plane(layers, pages, block, heads, pairs):
    gen = torch.Generator().manual_seed(pages)
    kv, sc = _runner_pool(gen, layers, pages, block, heads)
    order = torch.randperm(pages, generator=gen).tolist()
    src, dst = order[:pairs], order[pairs:2 * pairs]
    want = [_bytes(t).clone() for t in (kv, sc)]
    for w in want:
        w[:, :, dst] = w[:, :, src]
    M.copy_kv_blocks((kv, sc), src, dst, block_dim=2)
    for t, w in zip((kv, sc), want):
        assert torch.equal(_bytes(t), w)


def test_one_source_for_many_and_other_forms_of_the_ids():
    gen = torch.Generator().manual_seed(3)
    pool = torch.rand(10, 64, generator=gen).to(DEV)
    first = pool.clone()
    M.copy_kv_blocks(pool, torch.tensor([4, 4, 4]), np.array([1, 7, 9], np.int32))
    first[[1, 7, 9]] = first[4].clone()
    assert torch.equal(pool, first)
    M.copy_kv_blocks([pool], (1,), range(2, 3))
    assert torch.equal(pool[2], first[1])
    with pytest.raises(AssertionError, match="host"):
        M.copy_kv_blocks(pool, torch.tensor([4], device=DEV), [1])
    with pytest.raises(RuntimeError, match="not supported"):  # pages of 12 bytes
        M.copy_kv_blocks(torch.zeros(4, 3, device=DEV), [0], [1])


def test_pages_that_end_inside_a_segment_and_many_tensors():
    """Page sizes around the 16 KB that a workgroup takes, and more tensors
    than one launch holds."""
    gen = torch.Generator().manual_seed(4)
    pools = [torch.randint(0, 256, (2, 6, n), generator=gen, dtype=torch.uint8).to(DEV)
             for n in (16, 48, 4096, 16368, 16384, 16400, 32768, 50000, 112, 65552, 16)]
    want = [p.clone() for p in pools]
    for w in want:
        w[:, [5, 0, 3]] = w[:, [1, 2, 4]]
    M.copy_kv_blocks(pools, [1, 2, 4], [5, 0, 3], block_dim=1)
    for p, w in zip(pools, want):
        assert torch.equal(p, w)


def test_copies_of_a_pool_past_32_bits_of_bytes():
    pool = torch.empty(5, 1 << 30, dtype=torch.uint8, device=DEV)
    pool[4].fill_(9)
    pool[3, ::3] = 5
    M.copy_kv_blocks(pool, [4, 3], [0, 1])
    assert torch.equal(pool[0], pool[4]) and torch.equal(pool[1], pool[3])


def _plan(tables, n):
    """(remap, live, renamed tables, moves) of the documented rule."""
    used = {p for p in tables.flatten().tolist() if 0 <= p < n}
    named, live = sorted(used), len(used)
    holes = [p for p in range(live) if p not in used]
    remap = np.full(n, -1, np.int32)
    moves = []
    for p in named:
        remap[p] = p
        if p >= live:
            remap[p] = holes[len(moves)]
            moves.append((p, holes[len(moves)]))
    flat = [int(remap[p]) if 0 <= p < n else p for p in tables.flatten().tolist()]
    return remap, live, np.array(flat, np.int32).reshape(tables.shape), moves


def _check_compact(pools, tables, num_blocks, block_dim):
    before = [_bytes(p).clone() for p in pools]
    n = pools[0].shape[block_dim] if num_blocks is None else num_blocks
    remap, live, renamed, moves = _plan(tables, n)
    got_t, got_r, got_n = M.compact_kv_blocks(pools, torch.from_numpy(tables).to(DEV), num_blocks,
                                              block_dim=block_dim)
    np.testing.assert_array_equal(got_r.cpu().numpy(), remap)
    np.testing.assert_array_equal(got_t.cpu().numpy(), renamed)
    assert got_n.tolist() == [live]
    for p, b in zip(pools, before):
        b = b.movedim(block_dim, 0)
        want = b.clone()
        if moves:
            src, dst = zip(*moves)
            want[list(dst)] = b[list(src)]
        assert torch.equal(_bytes(p).movedim(block_dim, 0), want)


@pytest.mark.parametrize("pages,live,width", [
    (1, 1, 1), (1, 0, 1), (2, 1, 1), (31, 9, 4), (32, 32, 8), (33, 16, 5), (64, 1, 1),
    (65, 64, 9), (1000, 500, 40), (5000, 77, 100), (5000, 4999, 130), (70000, 30000, 200)])
def test_compaction_follows_the_rule(pages, live, width):
    gen = torch.Generator().manual_seed(pages + live)
    pool = torch.randint(0, 1 << 30, (2, pages, 8), generator=gen, dtype=torch.int32).to(DEV)
    for order in (torch.randperm(pages, generator=gen), torch.arange(pages).flip(0)):
        rows = -(-live // width) + 2
        tables = np.full((rows, width), -1, np.int32)
        tables.reshape(-1)[:live] = order[:live].numpy()
        tables[-1, 0] = tables[0, 0]  # a shared page
        _check_compact([pool], tables, None, 1)


def test_compaction_of_the_most_pages():
    """2^18 pages: the plan takes 98 KB of a workgroup's memory."""
    pages = 1 << 18
    gen = torch.Generator().manual_seed(15)
    pool = torch.randint(0, 1 << 30, (pages, 4), generator=gen, dtype=torch.int32).to(DEV)
    _check_compact([pool], torch.randperm(pages, generator=gen)[:90000].to(torch.int32).numpy()
                   .reshape(300, 300), None, 0)


def test_compaction_of_the_runners_pool_keeps_the_garbage_page():
    gen = torch.Generator().manual_seed(9)
    pools = _runner_pool(gen, 3, 21, 128, 4)
    tables = np.array([[19, 3, -1], [20, 7, 11], [3, 18, 25]], np.int32)  # 20: the garbage page
    before = _bytes(pools[0])[:, :, 20].clone()
    _check_compact(list(pools), tables, 20, 2)
    assert torch.equal(_bytes(pools[0])[:, :, 20], before)


def test_compaction_of_more_tensors_than_a_launch_and_of_no_table():
    gen = torch.Generator().manual_seed(10)
    pools = [torch.randint(0, 256, (12, 16 * (i + 1)), generator=gen, dtype=torch.uint8).to(DEV)
             for i in range(11)]
    _check_compact(pools, np.array([[11, 2, 9]], np.int32), None, 0)
    _check_compact(pools, np.zeros((0, 4), np.int32), None, 0)


def test_compaction_in_a_graph():
    gen = torch.Generator().manual_seed(12)
    pool = torch.randint(0, 256, (2, 300, 4096), generator=gen, dtype=torch.uint8).to(DEV)
    tables = torch.full((8, 20), -1, dtype=torch.int32, device=DEV)
    M.compact_kv_blocks(pool, tables, block_dim=1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        moved, remap, live = M.compact_kv_blocks(pool, tables, block_dim=1)
    for n in (100, 3, 160, 0):
        pages = torch.full((160,), -1, dtype=torch.int32)
        pages[:n] = torch.randperm(300, generator=gen)[:n].to(torch.int32)
        tables.copy_(pages.view(8, 20))
        before = pool.clone()
        graph.replay()
        torch.cuda.synchronize()
        r, count, renamed, moves = _plan(pages.view(8, 20).numpy(), 300)
        assert live.item() == count
        np.testing.assert_array_equal(remap.cpu().numpy(), r)
        np.testing.assert_array_equal(moved.cpu().numpy(), renamed)
        for src, dst in moves:
            before[:, dst] = before[:, src]
        assert torch.equal(pool, before)


def test_fork_of_both_formats():
    """A child's page reads as its parent's, in every layer, FP8 and 4 bits."""
    gen = torch.Generator().manual_seed(13)
    caches = M.allocate_fp4_kvcache(6, 128, 2, num_layers=3)
    key, value = (torch.randn(40, 2, 128, generator=gen).half().to(DEV) for _ in range(2))
    slots = torch.arange(40, device=DEV) + 2 * 128
    for i in range(3):
        M.store_fp4_kvcache(key * (i + 1), value, *(t[i] for t in caches), slots)
    M.copy_kv_blocks(caches, [2], [5], block_dim=1)
    for i in range(3):
        layer = tuple(t[i] for t in caches)
        a = M.load_fp4_kvcache(*layer, slots)
        b = M.load_fp4_kvcache(*layer, slots + 3 * 128)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and a[0].abs().sum() > 0


def test_native_paths_and_wrappers_agree(monkeypatch):
    """Every call above ran natively where it could; here the wrappers'."""
    from microserve_amd import _lib

    class Off:
        def __getattr__(self, name):
            return lambda *a: None

    gen = torch.Generator().manual_seed(14)
    first = list(_runner_pool(gen, 2, 30, 128, 2))
    other = [t.clone() for t in first]
    tables = torch.tensor([[29, 4, -1], [17, 28, 30]], dtype=torch.int32, device=DEV)
    assert _lib.fast.copy_blocks(tuple(first), [1, 2], (3, 4), 2) is True
    native = M.compact_kv_blocks(first, tables, 29, block_dim=2)
    assert _lib.fast.compact_blocks(first, tables, 29, 2) is not None
    for bad in (dict(src=[0, 1], dst=[2, 2]), dict(src=[3], dst=[3]), dict(src=[0], dst=[30])):
        with pytest.raises(AssertionError):
            M.copy_kv_blocks(first, bad["src"], bad["dst"], block_dim=2)
    with pytest.raises(AssertionError):
        M.compact_kv_blocks(first, tables, 31, block_dim=2)
    monkeypatch.setattr(_lib, "fast", Off())
    M.copy_kv_blocks(tuple(other), [1, 2], (3, 4), block_dim=2)
    for a, b in zip(native, M.compact_kv_blocks(other, tables, 29, block_dim=2)):
        assert torch.equal(a, b)
    M.compact_kv_blocks(other, tables, 29, block_dim=2)
    for a, b in zip(first, other):
        assert torch.equal(_bytes(a), _bytes(b))
