"""Attention weights of the FP8 cache's tokens, and eviction by them.

``weights`` is a fp32 tensor ``[NB, H_kv, BS]`` beside the caches
(``allocate_attention_weights``): a token's entry is the sum, over the q heads
that read its kv head and over queries, of the softmax probability that it got.
It is numbered by pages as the caches are, so ``copy_kv_blocks`` and
``compact_kv_blocks`` take it along.

``start`` (an integer, or an int32 tensor ``[B]``) is the first position that
takes part: a prefix whose pages several sequences share lies before it, is
never written and always stays.
"""

from __future__ import annotations

import torch

from microserve_amd import _lib


def allocate_attention_weights(num_blocks: int, block_size: int, num_kv_heads: int,
                               num_layers: int | None = None, device="cuda") -> torch.Tensor:
    """Zeroed ``weights``, with a leading layer dimension if ``num_layers`` is given."""
    shape = (num_blocks, num_kv_heads, block_size)
    lead = () if num_layers is None else (num_layers,)
    return torch.zeros(lead + shape, dtype=torch.float32, device=device)


def clear_attention_weights(weights: torch.Tensor, slot_mapping: torch.Tensor) -> None:
    """Set the entries of the tokens at ``slot_mapping`` (the store's: int32 or
    int64; slots outside the cache, -1 among them, are skipped) to 0.

    For the tokens that a prompt or a turn stores: a reused page, and the places
    behind ``evict_kv_tokens``'s lengths, hold the entries of what was there
    before.  ``Attention`` does this in its prefills.  Decode steps set their
    newest token's entry themselves, and so does a window without ``accumulate``.
    """
    what = "clear_attention_weights"
    assert weights.dim() == 3, f"{what}: weights must be [blocks, kv heads, block size]"
    _weights(what, weights, *weights.shape)
    assert slot_mapping.dtype in (torch.int32, torch.int64), (
        f"{what}: slot_mapping must be int32 or int64")
    slot_mapping = slot_mapping.contiguous()
    _lib.on_device(what, weights, slot_mapping)
    num_blocks, num_kv_heads, block_size = weights.shape
    with _lib.current(weights):
        status = _lib.load().mskv_clear_attention_weights(
            weights.data_ptr(), slot_mapping.data_ptr(),
            _lib.INT64 if slot_mapping.dtype == torch.int64 else _lib.INT32,
            slot_mapping.numel(), num_kv_heads, block_size, num_blocks, _lib.stream_of(weights))
    _lib.check(status, what)


def _start(what, start, batch, device):
    """(the int32 tensor or None, the integer)"""
    if isinstance(start, torch.Tensor):
        assert start.dtype == torch.int32 and start.numel() == batch, (
            f"{what}: start must be an integer or int32 [batch]")
        assert start.device == device, f"{what}: every tensor must be on {device}"
        return start.contiguous(), 0
    start = int(start)
    assert 0 <= start < 1 << 31, f"{what}: start must not be negative"
    return None, start


def _weights(what, weights, num_blocks, num_kv_heads, block_size):
    assert weights.dtype == torch.float32 and weights.is_contiguous(), (
        f"{what}: weights must be contiguous float32")
    assert tuple(weights.shape) == (num_blocks, num_kv_heads, block_size), (
        f"{what}: weights must be [blocks, kv heads, block size] = "
        f"{(num_blocks, num_kv_heads, block_size)}, got {tuple(weights.shape)}")


def _ptr(t):
    return None if t is None else t.data_ptr()


def _caches(what, k_cache, v_cache, k_scale_cache, v_scale_cache):
    assert k_cache.dtype == v_cache.dtype == torch.float8_e4m3fn
    assert k_scale_cache.dtype == v_scale_cache.dtype == torch.float32
    assert k_cache.dim() == 4 and v_cache.shape == k_cache.shape
    assert k_scale_cache.shape == v_scale_cache.shape == k_cache.shape[:3]
    for t in (k_cache, v_cache, k_scale_cache, v_scale_cache):
        assert t.is_contiguous(), f"{what}: caches must be contiguous"


def fp8_decode_attention_weights(
    query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
    k_scale_cache: torch.Tensor, v_scale_cache: torch.Tensor,
    cache_seqlens: torch.Tensor, block_tables: torch.Tensor, softmax_scale: float,
    weights: torch.Tensor, start: int | torch.Tensor = 0, out: torch.Tensor | None = None,
) -> torch.Tensor:
    """``fp8_decode_attention`` that also keeps its tokens' attention weights.

    The step's probabilities are added to the entries of ``weights``; the entry
    of the newest token, at position ``cache_seqlens - 1``, is set, so that it
    needs no clearing (a prompt's do: ``clear_attention_weights``).  Pages that two sequences of the batch
    name must lie before ``start``.  The call may be captured in a HIP graph.
    """
    res = _lib.fast.track(query, k_cache, v_cache, k_scale_cache, v_scale_cache, cache_seqlens,
                          block_tables, softmax_scale, weights, start, out)
    if res is not None:
        return res
    what = "fp8_decode_attention_weights"
    query = _lib.aligned(query)
    cache_seqlens, block_tables = cache_seqlens.contiguous(), block_tables.contiguous()
    assert query.dtype in (torch.float16, torch.bfloat16)
    _caches(what, k_cache, v_cache, k_scale_cache, v_scale_cache)
    batch, num_q_heads, head_dim = query.shape
    num_blocks, block_size, num_kv_heads = k_cache.shape[:3]
    assert cache_seqlens.dtype == block_tables.dtype == torch.int32
    assert num_q_heads % num_kv_heads == 0 and head_dim == k_cache.shape[3]
    assert block_tables.dim() == 2 and block_tables.shape[0] == batch == cache_seqlens.numel()
    _weights(what, weights, num_blocks, num_kv_heads, block_size)
    _lib.on_device(what, query, k_cache, v_cache, k_scale_cache, v_scale_cache, cache_seqlens,
                   block_tables, weights, out)
    starts, start = _start(what, start, batch, query.device)
    if out is None:
        out = torch.empty_like(query)
    else:
        assert out.shape == query.shape and out.dtype == query.dtype and out.is_contiguous()
    lib, width = _lib.load(), block_tables.shape[1]
    nbytes = lib.mskv_decode_weights_workspace_bytes(batch, num_q_heads, num_kv_heads, block_size,
                                                     width)
    with _lib.current(query):
        # on the current stream, as the prefill's partials are: reused in
        # stream order, and a graph's own under capture
        ws = torch.empty(nbytes, dtype=torch.uint8, device=query.device)
        status = lib.mskv_fp8_decode_attention_weights(
            query.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_scale_cache.data_ptr(),
            v_scale_cache.data_ptr(), cache_seqlens.data_ptr(), block_tables.data_ptr(),
            weights.data_ptr(), _ptr(starts), start, out.data_ptr(), batch, num_q_heads,
            num_kv_heads, head_dim, block_size, num_blocks, width, float(softmax_scale),
            _lib.act_dtype(query), ws.data_ptr(), nbytes, _lib.stream_of(query))
    _lib.check(status, what)
    return out


def fp8_window_attention_weights(
    query: torch.Tensor, k_cache: torch.Tensor, k_scale_cache: torch.Tensor,
    block_tables: torch.Tensor, cu_seqlens_q: torch.Tensor, cu_seqlens_k: torch.Tensor,
    max_seqlen_q: int, softmax_scale: float, weights: torch.Tensor, accumulate: bool = False,
    start: int | torch.Tensor = 0, max_seqlen_k: int | None = None,
) -> torch.Tensor:
    """The attention weights that each sequence's last queries give its tokens.

    ``query``, ``cu_seqlens_q`` and ``cu_seqlens_k`` describe the batch as for
    ``fp8_varlen_prefill_attention``: after a prompt, the last few rows of its
    queries, already stored tokens of the cache.  Query ``i`` of a sequence sees
    positions ``< Lk - Lq + i + 1``.  The entries of positions ``start .. Lk``
    are set (with ``accumulate``, added to: those of tokens that this turn has
    stored must have been cleared before, ``clear_attention_weights``); returns
    ``weights``.
    ``max_seqlen_q`` and ``max_seqlen_k`` (default: the tables' width) must be
    at least every sequence's numbers: what lies past them, or past the table,
    is not counted (``Lk`` stays the whole length).
    """
    res = _lib.fast.window(query, k_cache, k_scale_cache, block_tables, cu_seqlens_q, cu_seqlens_k,
                           max_seqlen_q, softmax_scale, weights, accumulate, start, max_seqlen_k)
    if res is not None:
        return res
    what = "fp8_window_attention_weights"
    query = _lib.aligned(query)
    block_tables = block_tables.contiguous()
    cu_seqlens_q, cu_seqlens_k = cu_seqlens_q.contiguous(), cu_seqlens_k.contiguous()
    assert query.dtype in (torch.float16, torch.bfloat16)
    _caches(what, k_cache, k_cache, k_scale_cache, k_scale_cache)
    total_q, num_q_heads, head_dim = query.shape
    num_blocks, block_size, num_kv_heads = k_cache.shape[:3]
    assert block_tables.dtype == cu_seqlens_q.dtype == cu_seqlens_k.dtype == torch.int32
    assert num_q_heads % num_kv_heads == 0 and head_dim == k_cache.shape[3]
    num_seqs = cu_seqlens_q.numel() - 1
    assert cu_seqlens_k.numel() == num_seqs + 1
    assert block_tables.dim() == 2 and block_tables.shape[0] == num_seqs
    _weights(what, weights, num_blocks, num_kv_heads, block_size)
    _lib.on_device(what, query, k_cache, k_scale_cache, block_tables, cu_seqlens_q, cu_seqlens_k,
                   weights)
    starts, start = _start(what, start, num_seqs, query.device)
    bound = 0 if max_seqlen_k is None else max(int(max_seqlen_k), 1)
    lib, width = _lib.load(), block_tables.shape[1]
    nbytes = lib.mskv_window_weights_bounded_workspace_bytes(
        total_q, int(max_seqlen_q), bound, num_q_heads, num_kv_heads, block_size, width)
    with _lib.current(query):
        ws = torch.empty(nbytes, dtype=torch.uint8, device=query.device)
        status = lib.mskv_fp8_window_attention_weights(
            query.data_ptr(), k_cache.data_ptr(), k_scale_cache.data_ptr(),
            block_tables.data_ptr(), cu_seqlens_q.data_ptr(), cu_seqlens_k.data_ptr(),
            weights.data_ptr(), _ptr(starts), start, int(bool(accumulate)), num_seqs, total_q,
            int(max_seqlen_q), bound, num_q_heads, num_kv_heads, head_dim, block_size, num_blocks,
            width, float(softmax_scale), _lib.act_dtype(query), ws.data_ptr(), nbytes,
            _lib.stream_of(query))
    _lib.check(status, what)
    return weights


def select_kv_tokens(weights: torch.Tensor, cache_seqlens: torch.Tensor,
                     block_tables: torch.Tensor, budget: int, recent: int = 0,
                     start: int | torch.Tensor = 0):
    """The tokens of every (sequence, kv head) that stay.

    Of ``L`` tokens ``n = min(L, budget)`` stay: the first ``start``, the last
    ``recent`` and the heaviest of those between (of equal weights the earlier
    one; a NaN counts as the lightest).  Where the first and the last ones do
    not all fit, the first ones go before.  Returns ``(kept, seqlens)``: int32
    ``[B, H_kv, budget]``, the positions that stay in ascending order and -1
    behind them, and int32 ``[B]``, ``n``.  Any fp32 ``[NB, H_kv, BS]`` serves
    as ``weights``.  Nothing is read on the host.
    """
    res = _lib.fast.choose(weights, cache_seqlens, block_tables, budget, recent, start)
    if res is not None:
        return res
    what = "select_kv_tokens"
    assert weights.dim() == 3, f"{what}: weights must be [blocks, kv heads, block size]"
    num_blocks, num_kv_heads, block_size = weights.shape
    _weights(what, weights, num_blocks, num_kv_heads, block_size)
    cache_seqlens, block_tables = cache_seqlens.contiguous(), block_tables.contiguous()
    assert cache_seqlens.dtype == block_tables.dtype == torch.int32
    batch = cache_seqlens.numel()
    assert block_tables.dim() == 2 and block_tables.shape[0] == batch
    budget, recent = int(budget), int(recent)
    assert 0 < budget < 1 << 31, f"{what}: budget must be positive"
    assert 0 <= recent < 1 << 31, f"{what}: recent must not be negative"
    _lib.on_device(what, weights, cache_seqlens, block_tables)
    starts, start = _start(what, start, batch, weights.device)
    with _lib.current(weights):
        ints = dict(dtype=torch.int32, device=weights.device)
        kept = torch.empty(batch, num_kv_heads, budget, **ints)
        seqlens = torch.empty(batch, **ints)
        status = _lib.load().mskv_select_kv_tokens(
            weights.data_ptr(), cache_seqlens.data_ptr(), block_tables.data_ptr(), _ptr(starts),
            start, recent, budget, kept.data_ptr(), seqlens.data_ptr(), batch, num_kv_heads,
            block_size, num_blocks, block_tables.shape[1], _lib.stream_of(weights))
    _lib.check(status, what)
    return kept, seqlens


def evict_kv_tokens(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale_cache: torch.Tensor,
                    v_scale_cache: torch.Tensor, kept: torch.Tensor, seqlens: torch.Tensor,
                    block_tables: torch.Tensor, weights: torch.Tensor | None = None) -> None:
    """Move the kept tokens together, in place: position ``i`` of every
    (sequence, kv head) gets the row, the scales and, if ``weights`` is given,
    the weight of position ``kept[b, h, i]``, for ``i < seqlens[b]``.

    ``kept`` and ``seqlens`` are ``select_kv_tokens``'s (``kept`` must ascend).
    Keys carry their rotary embedding from before they were stored, so the
    sequence goes on at its own positions over a cache of ``seqlens`` tokens:
    the next token's slot and length follow ``seqlens``, its rotary position
    does not.  Pages behind ``seqlens`` are free to give back.  A page whose
    rows move must belong to one sequence alone: copy a shared one first
    (``copy_kv_blocks``), or keep it before ``start``.  The same rows of several
    layers take a call each.
    """
    if _lib.fast.evict(k_cache, v_cache, k_scale_cache, v_scale_cache, kept, seqlens, block_tables,
                       weights):
        return
    what = "evict_kv_tokens"
    _caches(what, k_cache, v_cache, k_scale_cache, v_scale_cache)
    num_blocks, block_size, num_kv_heads, head_dim = k_cache.shape
    assert kept.dtype == seqlens.dtype == block_tables.dtype == torch.int32
    batch = seqlens.numel()
    assert kept.dim() == 3 and kept.shape[:2] == (batch, num_kv_heads), (
        f"{what}: kept must be [batch, kv heads, budget]")
    assert block_tables.dim() == 2 and block_tables.shape[0] == batch
    if weights is not None:
        _weights(what, weights, num_blocks, num_kv_heads, block_size)
    kept, seqlens, block_tables = kept.contiguous(), seqlens.contiguous(), block_tables.contiguous()
    _lib.on_device(what, k_cache, v_cache, k_scale_cache, v_scale_cache, kept, seqlens,
                   block_tables, weights)
    with _lib.current(k_cache):
        status = _lib.load().mskv_evict_kv_tokens(
            k_cache.data_ptr(), v_cache.data_ptr(), k_scale_cache.data_ptr(),
            v_scale_cache.data_ptr(), _ptr(weights), kept.data_ptr(), seqlens.data_ptr(),
            block_tables.data_ptr(), batch, num_kv_heads, head_dim, block_size, num_blocks,
            block_tables.shape[1], kept.shape[2], _lib.stream_of(k_cache))
    _lib.check(status, what)
