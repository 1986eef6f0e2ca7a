"""Moving the pages of a paged KV pool: copies to other pages (a forked
sequence's last page, copy-on-write) and compaction, in every layer and plane
in one launch, over FP8 and 4-bit caches alike."""

from __future__ import annotations

import ctypes
from array import array

import torch

from microserve_amd import _lib

MAX_POOLS = 8  # tensors of one launch (MSKV_MAX_POOLS)


def _tensors(caches):
    return (caches,) if isinstance(caches, torch.Tensor) else tuple(caches)


def _pools(what, caches, block_dim):
    """Checks the caches of a call; their host descriptions, at most MAX_POOLS
    each, and the number of blocks."""
    assert caches, f"{what}: no caches"
    assert block_dim >= 0
    num_blocks = None
    _lib.on_device(what, *caches)
    rows = []
    for t in caches:
        assert t.is_contiguous(), "caches must be contiguous"
        assert t.dim() > block_dim, f"{what}: dimension {block_dim} must number the blocks"
        n = t.shape[block_dim]
        assert num_blocks in (None, n), f"{what}: every cache must have the same blocks"
        num_blocks = n
        planes = 1
        for size in t.shape[:block_dim]:
            planes *= size
        assert t.numel() > 0, f"{what}: an empty cache"
        page = t.numel() // (planes * n) * t.element_size()
        rows.append((t.data_ptr(), planes, n * page, page))
    groups = []
    for at in range(0, len(rows), MAX_POOLS):
        part = rows[at:at + MAX_POOLS]
        n = len(part)
        groups.append((n, (ctypes.c_void_p * n)(*(r[0] for r in part)),
                       *((ctypes.c_int64 * n)(*(r[i] for r in part)) for i in (1, 2, 3))))
    return groups, num_blocks


def _check_all(what, lib, groups, num_blocks, compact):
    """Refuses a pool of several launches before the first of them."""
    if len(groups) > 1:
        for count, *described in groups:
            _lib.check(lib.mskv_check_kv_blocks(count, *described, num_blocks, compact), what)


def _ids(what, blocks):
    if isinstance(blocks, torch.Tensor):
        assert not blocks.is_cuda, f"{what}: block ids are host integers"
        assert blocks.dtype in (torch.int32, torch.int64)
        blocks = blocks.flatten().tolist()
    try:
        return array("i", blocks)
    except OverflowError as e:
        raise AssertionError(f"{what}: a block id is out of range") from e


def copy_kv_blocks(caches, src_blocks, dst_blocks, block_dim: int = 0) -> None:
    """Copy pages: in every cache, ``page[dst_blocks[i]] = page[src_blocks[i]]``.

    ``caches`` is a tensor or a sequence of them whose dimension ``block_dim``
    numbers the pages: the runner's ``[2, L, NB + 1, ...]`` caches and scales
    with ``block_dim=2``, one layer's caches with 0.  The ids are host
    integers (the block manager's), a list or a CPU tensor, and travel with
    the launch.  No page may be written twice or be both read and written
    (AssertionError), so the order of the pairs does not matter.  Tensors start
    and pages end on 16 bytes (RuntimeError); a call that is refused has moved
    nothing.

    To fork a sequence, give the child the parent's full pages and copy the
    partly filled one to a page of its own.
    """
    if _lib.fast.copy_blocks(caches, src_blocks, dst_blocks, block_dim):
        return
    what = "copy_kv_blocks"
    src, dst = _ids(what, src_blocks), _ids(what, dst_blocks)
    assert len(src) == len(dst), f"{what}: as many destinations as sources"
    tensors = _tensors(caches)
    groups, num_blocks = _pools(what, tensors, block_dim)
    if not src:
        return
    for ids in (src, dst):
        assert min(ids) >= 0 and max(ids) < num_blocks, f"{what}: block ids must lie in the pool"
    written = set(dst)
    assert len(written) == len(dst), f"{what}: a block is written twice"
    assert written.isdisjoint(src), f"{what}: a block is both read and written"
    src_at, dst_at = src.buffer_info()[0], dst.buffer_info()[0]
    lib = _lib.load()
    _check_all(what, lib, groups, num_blocks, compact=0)
    with _lib.current(tensors[0]):
        stream = _lib.stream_of(tensors[0])
        for count, *described in groups:
            _lib.check(lib.mskv_copy_kv_blocks(count, *described, num_blocks, src_at, dst_at,
                                               len(src), stream), what)


def compact_kv_blocks(caches, block_tables: torch.Tensor, num_blocks: int | None = None,
                      block_dim: int = 0):
    """Move the pages that ``block_tables`` names to the pool's lowest places.

    Returns ``(block_tables, remap, num_live)``: the int32 tables with their
    entries renamed (a new tensor), each page's new place (int32
    ``[num_blocks]``, -1 for a page that no entry names) and the number of
    live pages (int32 ``[1]``), which fill places ``0 .. num_live - 1``.  A
    live page below ``num_live`` stays; the others take the free places in
    ascending order.

    A page that no entry names is free to this call and may be overwritten.
    Pages that are cached without a running sequence (a prefix cache's) must
    be named too, in rows of their own, and whatever else holds page numbers
    (the hash table of cached pages, reference counts, the free list, the
    sequences' own tables) must be renamed by ``remap`` before it is used again.

    ``num_blocks`` is the number of pages that take part, the first ones of
    dimension ``block_dim`` (default: all); entries outside them (-1 padding,
    the runner's garbage page behind the pool) are kept as they are.  Nothing
    is read on the host, and the call may be captured in a HIP graph.  Refusals
    are ``copy_kv_blocks``'s, and more than 2^18 pages; they come before any
    page moves.
    """
    res = _lib.fast.compact_blocks(caches, block_tables, num_blocks, block_dim)
    if res is not None:
        return res
    what = "compact_kv_blocks"
    tensors = _tensors(caches)
    groups, pool = _pools(what, tensors, block_dim)
    num_blocks = pool if num_blocks is None else int(num_blocks)
    assert 0 < num_blocks <= pool, f"{what}: num_blocks must lie in the pool"
    assert block_tables.dtype == torch.int32
    _lib.on_device(what, tensors[0], block_tables)
    tables = block_tables.contiguous()
    lib = _lib.load()
    _check_all(what, lib, groups, num_blocks, compact=1)
    with _lib.current(tables):
        ints = dict(dtype=torch.int32, device=tables.device)
        renamed = torch.empty(tables.shape, **ints)
        remap, live = torch.empty(num_blocks, **ints), torch.empty(1, **ints)
        stream = _lib.stream_of(tables)
        for count, *described in groups:
            # (a later group's plan is the first one's: the tables are kept)
            _lib.check(lib.mskv_compact_kv_blocks(
                count, *described, num_blocks, tables.data_ptr(), tables.numel(),
                renamed.data_ptr(), remap.data_ptr(), live.data_ptr(), stream), what)
    return renamed, remap, live
