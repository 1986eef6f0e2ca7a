"""Decode attention for sequences that share prefixes (requests that hit the
block manager's prefix cache, samples of one prompt, forks): the shared pages
are read once for a whole group."""

from __future__ import annotations

import torch

from microserve_amd import _lib

MAX_GROUPS = 1024


def group_by_prefix(block_tables, block_size: int):
    """Groups of sequences that name the same first pages.

    ``block_tables`` is the sequences' lists of pages (the block manager's).
    Returns ``(order, cu_groups, prefix_lens)``, lists of host integers: the
    order in which the batch must be built so that a group's sequences follow
    one another, the groups' boundaries in it, and the tokens of each group's
    shared pages.  Sequences that share their first page are one group, and its
    prefix is what all of them share; a sequence alone has a prefix of 0.
    """
    tables = [list(t) for t in block_tables]
    order = sorted(range(len(tables)), key=lambda i: (tables[i][:1], i))
    cu, prefixes = [0], []
    for at, i in enumerate(order):
        first = tables[order[cu[-1]]]
        if at > cu[-1] and tables[i][:1] == first[:1] and first:
            same = min(prefixes[-1], len(tables[i]))
            prefixes[-1] = next((j for j in range(same) if tables[i][j] != first[j]), same)
            continue
        if at:
            cu.append(at)
        prefixes.append(len(tables[i]))
    if order:
        cu.append(len(order))
    alone = [b - a == 1 for a, b in zip(cu, cu[1:])]
    return order, cu, [0 if one else n * block_size for one, n in zip(alone, prefixes)]


def fp8_shared_prefix_decode_attention(
    query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
    k_scale_cache: torch.Tensor, v_scale_cache: torch.Tensor,
    cache_seqlens: torch.Tensor, block_tables: torch.Tensor, softmax_scale: float,
    cu_groups: torch.Tensor, prefix_lens: torch.Tensor, max_prefix_len: int | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """``fp8_decode_attention`` where groups of sequences share their first pages.

    The first ``prefix_lens[g]`` tokens of sequences ``cu_groups[g]`` to
    ``cu_groups[g + 1] - 1`` lie in the same pages (int32 tensors on the GPU,
    ``cu_groups`` ascending).  ``cache_seqlens`` and ``block_tables`` describe
    whole contexts, as for ``fp8_decode_attention``, and the result is that
    call's.  ``max_prefix_len``, a host integer, is the longest prefix that is
    read once (default: the tables' width); what a group shares beyond it, past
    its shortest sequence or past a multiple of 128 tokens is read sequence by
    sequence.  The launch depends on shapes and ``max_prefix_len`` alone, so the
    call can be captured in a HIP graph.
    """
    res = _lib.fast.shared(query, k_cache, v_cache, k_scale_cache, v_scale_cache, cache_seqlens,
                           block_tables, softmax_scale, cu_groups, prefix_lens, max_prefix_len,
                           out)
    if res is not None:
        return res
    what = "fp8_shared_prefix_decode_attention"
    query = _lib.aligned(query)
    cache_seqlens, block_tables = cache_seqlens.contiguous(), block_tables.contiguous()
    cu_groups, prefix_lens = cu_groups.contiguous(), prefix_lens.contiguous()
    batch, num_q_heads, head_dim = query.shape
    assert query.dtype in (torch.float16, torch.bfloat16)
    assert k_cache.dtype == v_cache.dtype == torch.float8_e4m3fn
    assert k_scale_cache.dtype == v_scale_cache.dtype == torch.float32
    assert k_cache.dim() == 4 and v_cache.shape == k_cache.shape
    assert k_scale_cache.shape == v_scale_cache.shape == k_cache.shape[:3]
    for t in (k_cache, v_cache, k_scale_cache, v_scale_cache):
        assert t.is_contiguous(), "caches must be contiguous"
    num_blocks, block_size, num_kv_heads = k_cache.shape[:3]
    for t in (cache_seqlens, block_tables, cu_groups, prefix_lens):
        assert t.dtype == torch.int32
    assert num_q_heads % num_kv_heads == 0 and head_dim == k_cache.shape[3]
    assert block_tables.dim() == 2 and block_tables.shape[0] == batch == cache_seqlens.numel()
    groups = prefix_lens.numel()
    assert cu_groups.numel() == groups + 1, f"{what}: cu_groups must be [groups + 1]"
    assert groups <= MAX_GROUPS, f"{what}: at most {MAX_GROUPS} groups"
    _lib.on_device(what, query, k_cache, v_cache, k_scale_cache, v_scale_cache, cache_seqlens,
                   block_tables, cu_groups, prefix_lens, out)
    width = block_tables.shape[1]
    bound = width * block_size if max_prefix_len is None else int(max_prefix_len)
    assert bound >= 0, f"{what}: max_prefix_len must not be negative"
    if out is None:
        out = torch.empty_like(query)
    else:
        assert out.shape == query.shape and out.dtype == query.dtype and out.is_contiguous()
    lib = _lib.load()
    nbytes = lib.mskv_shared_decode_workspace_bytes(batch, groups, num_q_heads, num_kv_heads,
                                                    block_size, width, bound)
    with _lib.current(query):
        # on the current stream: reused in stream order, and a graph's own
        # under capture
        ws = torch.empty(nbytes, dtype=torch.uint8, device=query.device)
        status = lib.mskv_fp8_shared_prefix_decode_attention(
            query.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_scale_cache.data_ptr(),
            v_scale_cache.data_ptr(), cache_seqlens.data_ptr(), block_tables.data_ptr(),
            cu_groups.data_ptr(), prefix_lens.data_ptr(), bound, out.data_ptr(), batch, groups,
            num_q_heads, num_kv_heads, head_dim, block_size, num_blocks, width,
            float(softmax_scale), _lib.act_dtype(query), ws.data_ptr(), nbytes,
            _lib.stream_of(query))
    _lib.check(status, what)
    return out
