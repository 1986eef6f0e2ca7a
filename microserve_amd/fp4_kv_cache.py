"""The 4-bit paged KV cache: allocation, quantizing store and read-back,
backed by the gfx950 HIP kernels.

A value is an e2m1 code (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign), two to a
byte.  K carries a power-of-two scale for each 32 dimensions of a (token, kv
head) row, V one fp32 scale a row: 136 bytes a token and kv head, against 264
of the FP8 cache.  The pages of K lie in the matrix unit's operand order:

    k_cache        uint8 [NB, H_kv, BS / 16, 4, 16, 16]
    v_cache        uint8 [NB, H_kv, BS, 64]
    k_scale_cache  uint8 [NB, H_kv, BS / 64, 4, 16, 4]
    v_scale_cache  fp32  [NB, H_kv, BS]
"""

from __future__ import annotations

import torch

from microserve_amd import _lib

FP4_MAX = 6.0
HEAD_DIM = 128
BLOCK_UNIT = 128  # block sizes are multiples of it


def fp4_cache_shapes(num_blocks: int, block_size: int, num_kv_heads: int):
    """The shapes of ``(k_cache, v_cache, k_scale_cache, v_scale_cache)``."""
    assert block_size > 0 and block_size % BLOCK_UNIT == 0, (
        f"block_size must be a multiple of {BLOCK_UNIT}, got {block_size}")
    nb, h, bs = num_blocks, num_kv_heads, block_size
    return ((nb, h, bs // 16, 4, 16, 16), (nb, h, bs, 64), (nb, h, bs // 64, 4, 16, 4), (nb, h, bs))


def allocate_fp4_kvcache(num_blocks: int, block_size: int, num_kv_heads: int,
                         num_layers: int | None = None, device="cuda"):
    """Zeroed ``(k_cache, v_cache, k_scale_cache, v_scale_cache)``.

    With ``num_layers`` each tensor has a leading layer dimension: layer
    ``i``'s caches are ``tuple(t[i] for t in caches)``, as the runner injects
    per-layer views of its own (``model_runner.py:111-122``).
    """
    shapes = fp4_cache_shapes(num_blocks, block_size, num_kv_heads)
    lead = () if num_layers is None else (num_layers,)
    types = (torch.uint8, torch.uint8, torch.uint8, torch.float32)
    return tuple(torch.zeros(lead + s, dtype=t, device=device) for s, t in zip(shapes, types))


def check_fp4_caches(k_cache, v_cache, k_scale_cache, v_scale_cache):
    """``(num_blocks, num_kv_heads, block_size)`` of a layer's four caches."""
    assert v_cache.dim() == 4 and v_cache.shape[3] == HEAD_DIM // 2, (
        f"v_cache must be [blocks, kv heads, block size, {HEAD_DIM // 2}], got "
        f"{tuple(v_cache.shape)}")
    num_blocks, num_kv_heads, block_size = v_cache.shape[:3]
    shapes = fp4_cache_shapes(num_blocks, block_size, num_kv_heads)
    for name, t, shape, dtype in zip(
            ("k_cache", "v_cache", "k_scale_cache", "v_scale_cache"),
            (k_cache, v_cache, k_scale_cache, v_scale_cache), shapes,
            (torch.uint8, torch.uint8, torch.uint8, torch.float32)):
        assert t.dtype == dtype and tuple(t.shape) == shape, (
            f"{name} must be {dtype} {shape}, got {t.dtype} {tuple(t.shape)}")
        assert t.is_contiguous(), "caches must be contiguous"
    return num_blocks, num_kv_heads, block_size


def _slots(slot_mapping):
    assert slot_mapping.dtype in (torch.int32, torch.int64)
    return slot_mapping.contiguous(), (
        _lib.INT64 if slot_mapping.dtype == torch.int64 else _lib.INT32)


def store_fp4_kvcache(
    key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor,
    v_cache: torch.Tensor, k_scale_cache: torch.Tensor,
    v_scale_cache: torch.Tensor, slot_mapping: torch.Tensor,
) -> None:
    """Quantize ``key``/``value`` rows and write them at ``slot_mapping``.

    ``store_fp8_kvcache``'s arguments over the 4-bit cache.  Token ``t`` lands
    in slot ``slot_mapping[t]``: token ``slot % BS`` of block ``slot // BS``;
    slots outside the cache are skipped, and one that several tokens name (as
    the runner's padding does its garbage slot) holds unspecified bytes.  K's
    scale is the power of two, for each 32 dimensions, that brings the largest
    magnitude to at most 7 (a 7 rounds to 6, half of the last step); V's is
    ``max(amax, 1e-8) / 6``.  Codes are nearest, ties to even.  32 dimensions
    of K, or a row of V, that hold an infinity or a NaN read back as NaN.
    """
    if _lib.fast.store4(key, value, k_cache, v_cache, k_scale_cache, v_scale_cache,
                        slot_mapping):
        return
    num_blocks, num_kv_heads, block_size = check_fp4_caches(
        k_cache, v_cache, k_scale_cache, v_scale_cache)
    assert key.dim() == 3 and value.shape == key.shape
    assert value.dtype == key.dtype
    assert key.shape[1:] == (num_kv_heads, HEAD_DIM)
    slots, slot_type = _slots(slot_mapping)
    assert slots.numel() == key.shape[0]
    _lib.on_device("store_fp4_kvcache", key, value, k_cache, v_cache, k_scale_cache,
                   v_scale_cache, slots)
    key, key_stride = _lib.token_rows(key)
    value, value_stride = _lib.token_rows(value)
    with _lib.current(key):
        status = _lib.load().mskv_store_fp4_kvcache(
            key.data_ptr(), key_stride, value.data_ptr(), value_stride, k_cache.data_ptr(),
            v_cache.data_ptr(), k_scale_cache.data_ptr(), v_scale_cache.data_ptr(),
            slots.data_ptr(), slot_type, key.shape[0], num_kv_heads, HEAD_DIM, block_size,
            num_blocks, _lib.store_dtype(key), _lib.stream_of(key))
    _lib.check(status, "store_fp4_kvcache")


def load_fp4_kvcache(
    k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale_cache: torch.Tensor,
    v_scale_cache: torch.Tensor, slot_mapping: torch.Tensor,
    dtype: torch.dtype = torch.bfloat16,
) -> tuple[torch.Tensor, torch.Tensor]:
    """The keys and values that the slots hold, ``[tokens, H_kv, D]`` each:
    ``code * scale`` rounded to ``dtype`` (fp16, bf16 or fp32).  Zeros for
    slots outside the cache."""
    res = _lib.fast.load4(k_cache, v_cache, k_scale_cache, v_scale_cache, slot_mapping, dtype)
    if res is not None:
        return res
    num_blocks, num_kv_heads, block_size = check_fp4_caches(
        k_cache, v_cache, k_scale_cache, v_scale_cache)
    slots, slot_type = _slots(slot_mapping)
    _lib.on_device("load_fp4_kvcache", slots, k_cache, v_cache, k_scale_cache, v_scale_cache)
    key = torch.empty(slots.numel(), num_kv_heads, HEAD_DIM, dtype=dtype, device=slots.device)
    value = torch.empty_like(key)
    with _lib.current(key):
        status = _lib.load().mskv_load_fp4_kvcache(
            k_cache.data_ptr(), v_cache.data_ptr(), k_scale_cache.data_ptr(),
            v_scale_cache.data_ptr(), slots.data_ptr(), slot_type, key.data_ptr(),
            value.data_ptr(), slots.numel(), num_kv_heads, HEAD_DIM, block_size, num_blocks,
            _lib.store_dtype(key), _lib.stream_of(key))
    _lib.check(status, "load_fp4_kvcache")
    return key, value
