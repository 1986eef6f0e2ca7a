"""Decode and causal chunk / varlen prefill attention over the 4-bit paged KV
cache (``fp4_kv_cache``), backed by the gfx950 HIP kernels."""

from __future__ import annotations

import torch

from microserve_amd import _lib
from microserve_amd.fp4_kv_cache import HEAD_DIM, check_fp4_caches
from microserve_amd.fp8_decode_attention import _scratch


def _check(what, query, caches):
    num_blocks, num_kv_heads, block_size = check_fp4_caches(*caches)
    assert query.dim() == 3 and query.shape[2] == HEAD_DIM
    assert query.dtype in (torch.float16, torch.bfloat16)
    assert query.shape[1] % num_kv_heads == 0
    _lib.on_device(what, query, *caches)
    return num_blocks, num_kv_heads, block_size


def fp4_decode_attention(
    query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
    k_scale_cache: torch.Tensor, v_scale_cache: torch.Tensor,
    cache_seqlens: torch.Tensor, block_tables: torch.Tensor,
    softmax_scale: float, out: torch.Tensor | None = None,
) -> torch.Tensor:
    """One decode step: ``query`` ``[B, H_q, D]`` against the 4-bit cache.

    ``fp8_decode_attention``'s arguments and rules: rows of length 0 are
    zeros, block ids outside the pool read as empty, the split count depends
    on shapes only and the split partials live in the persistent scratch of
    the (device, stream), so the call may be captured in a HIP graph; graphs
    captured on one stream share that scratch and replay one after the other.
    """
    res = _lib.fast.decode4(query, k_cache, v_cache, k_scale_cache, v_scale_cache, cache_seqlens,
                            block_tables, softmax_scale, out, _scratch)
    if res is not None:
        return res
    query = _lib.aligned(query)
    cache_seqlens = cache_seqlens.contiguous()
    block_tables = block_tables.contiguous()
    num_blocks, num_kv_heads, block_size = _check(
        "fp4_decode_attention", query, (k_cache, v_cache, k_scale_cache, v_scale_cache))
    batch_size, num_q_heads, head_dim = query.shape
    assert cache_seqlens.dtype == torch.int32
    assert block_tables.dtype == torch.int32 and block_tables.dim() == 2
    assert block_tables.shape[0] == batch_size == cache_seqlens.numel()
    _lib.on_device("fp4_decode_attention", query, cache_seqlens, block_tables, out)
    if out is None:
        out = torch.empty_like(query)
    else:
        assert out.shape == query.shape and out.dtype == query.dtype and out.is_contiguous()
    lib = _lib.load()
    width = block_tables.shape[1]
    splits = lib.mskv_fp4_decode_num_splits(batch_size, num_q_heads, num_kv_heads, width,
                                            block_size)
    ws_bytes = lib.mskv_decode_workspace_bytes(batch_size, num_q_heads, num_kv_heads, head_dim,
                                               splits)
    with _lib.current(query):
        stream = _lib.stream_of(query)
        ws = _scratch(query.device, stream, ws_bytes) if ws_bytes else None
        status = lib.mskv_fp4_decode_attention(
            query.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_scale_cache.data_ptr(),
            v_scale_cache.data_ptr(), cache_seqlens.data_ptr(), block_tables.data_ptr(),
            out.data_ptr(), batch_size, num_q_heads, num_kv_heads, head_dim, block_size,
            num_blocks, width, float(softmax_scale), _lib.act_dtype(query), splits,
            None if ws is None else ws.data_ptr(), ws_bytes, stream)
    _lib.check(status, "fp4_decode_attention")
    return out


def _launch(what, query, caches, dims, tables, cu_q, cu_k, prefix_len, num_seqs, max_seqlen_q,
            max_seqlen_k, width, softmax_scale):
    num_blocks, num_kv_heads, block_size = dims
    total_q, num_q_heads, head_dim = query.shape
    lib = _lib.load()
    output = torch.empty_like(query)
    if total_q == 0 or num_seqs == 0:
        return output
    ws_bytes = lib.mskv_fp8_prefill_bounded_workspace_bytes(
        num_seqs, total_q, max_seqlen_q, max_seqlen_k, num_q_heads, num_kv_heads, head_dim,
        block_size, width)
    with _lib.current(query):
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=query.device) if ws_bytes else None
        status = lib.mskv_fp4_prefill_attention(
            query.data_ptr(), *(t.data_ptr() for t in caches), tables.data_ptr(),
            None if cu_q is None else cu_q.data_ptr(), None if cu_k is None else cu_k.data_ptr(),
            prefix_len, output.data_ptr(), num_seqs, total_q, max_seqlen_q, max_seqlen_k,
            num_q_heads, num_kv_heads, head_dim, block_size, num_blocks, width,
            float(softmax_scale), _lib.act_dtype(query), None if ws is None else ws.data_ptr(),
            ws_bytes, _lib.stream_of(query))
    _lib.check(status, what)
    return output


def fp4_chunk_prefill_attention(
    query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
    k_scale_cache: torch.Tensor, v_scale_cache: torch.Tensor,
    block_table: torch.Tensor, prefix_len: int, softmax_scale: float,
) -> torch.Tensor:
    """Single-sequence causal chunk prefill over the 4-bit cache:
    ``fp8_chunk_prefill_attention``'s arguments.  Query ``i`` of the chunk
    sees the cached positions ``< prefix_len + i + 1``."""
    res = _lib.fast.prefill4(query, k_cache, v_cache, k_scale_cache, v_scale_cache, block_table,
                             None, None, prefix_len, 0, 0, softmax_scale)
    if res is not None:
        return res
    query = _lib.aligned(query)
    block_table = block_table.contiguous().view(-1)
    caches = (k_cache, v_cache, k_scale_cache, v_scale_cache)
    dims = _check("fp4_chunk_prefill_attention", query, caches)
    assert block_table.dtype == torch.int32
    _lib.on_device("fp4_chunk_prefill_attention", query, block_table)
    prefix_len = int(prefix_len)
    assert prefix_len >= 0
    n = query.shape[0]
    return _launch("fp4_chunk_prefill_attention", query, caches, dims, block_table, None, None,
                   prefix_len, 1, n, prefix_len + n, block_table.numel(), softmax_scale)


def fp4_varlen_prefill_attention(
    query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
    k_scale_cache: torch.Tensor, v_scale_cache: torch.Tensor,
    block_tables: torch.Tensor, cu_seqlens_q: torch.Tensor,
    cu_seqlens_k: torch.Tensor, max_seqlen_q: int, softmax_scale: float,
    max_seqlen_k: int | None = None,
) -> torch.Tensor:
    """Varlen causal prefill with cached prefixes over the 4-bit cache, in one
    launch: ``fp8_varlen_prefill_attention``'s arguments.  Rows of ``query``
    behind the last sequence, and rows past ``max_seqlen_q`` of their
    sequence, are not written."""
    bound = 0 if max_seqlen_k is None else int(max_seqlen_k)
    res = _lib.fast.prefill4(query, k_cache, v_cache, k_scale_cache, v_scale_cache, block_tables,
                             cu_seqlens_q, cu_seqlens_k, 0, max_seqlen_q, bound, softmax_scale)
    if res is not None:
        return res
    query = _lib.aligned(query)
    block_tables = block_tables.contiguous()
    cu_seqlens_q = cu_seqlens_q.contiguous()
    cu_seqlens_k = cu_seqlens_k.contiguous()
    caches = (k_cache, v_cache, k_scale_cache, v_scale_cache)
    dims = _check("fp4_varlen_prefill_attention", query, caches)
    assert block_tables.dtype == cu_seqlens_q.dtype == cu_seqlens_k.dtype == torch.int32
    num_seqs = cu_seqlens_q.numel() - 1
    assert cu_seqlens_k.numel() == num_seqs + 1
    assert block_tables.dim() == 2 and block_tables.shape[0] == num_seqs
    _lib.on_device("fp4_varlen_prefill_attention", query, block_tables, cu_seqlens_q,
                   cu_seqlens_k)
    return _launch("fp4_varlen_prefill_attention", query, caches, dims, block_tables,
                   cu_seqlens_q, cu_seqlens_k, 0, num_seqs, int(max_seqlen_q), max(bound, 0),
                   block_tables.shape[1], softmax_scale)
