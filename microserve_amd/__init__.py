"""MI355X-native FP8 paged-KV hot path of microserve.

Drop-in replacements for ``microserve.layers.fp8_kv_cache``,
``fp8_decode_attention``, ``fp8_chunk_prefill_attention``, the fresh-prefill
``flash_attn_varlen_func`` call,
``layers.attention.Attention`` (FP8 branch), ``utils.context``, the runner's
step-input builders (``step_inputs``) and the fused q/k norm + rotary + store
prologue (``qk_norm_rope_store``), backed by
hand-written gfx950 HIP kernels behind the C ABI in ``include/mskv.h``.

Beside them, the same path over a cache held in 4 bits (``fp4_kv_cache``,
``fp4_attention``; the ``Attention`` layer takes either), the moving of a
pool's pages (``kv_blocks``), the decode of sequences that share prefixes
(``shared_prefix``), and the attention weights of cached tokens with
eviction by them (``attention_weights``).
"""

from microserve_amd.context import (  # noqa: F401
    AttentionMode, Context, get_context, reset_context, set_context)
from microserve_amd.fp8_kv_cache import store_fp8_kvcache  # noqa: F401
from microserve_amd.fp8_decode_attention import (  # noqa: F401
    decode_num_splits, fp8_decode_attention)
from microserve_amd.fp8_chunk_prefill_attention import (  # noqa: F401
    fp8_chunk_prefill_attention, fp8_varlen_prefill_attention)
from microserve_amd.varlen_attention import (  # noqa: F401
    flash_attn_varlen_func, varlen_attention)
from microserve_amd.qk_norm_rope import qk_norm_rope_store  # noqa: F401
from microserve_amd.fp4_kv_cache import (  # noqa: F401
    allocate_fp4_kvcache, fp4_cache_shapes, load_fp4_kvcache, store_fp4_kvcache)
from microserve_amd.fp4_attention import (  # noqa: F401
    fp4_chunk_prefill_attention, fp4_decode_attention, fp4_varlen_prefill_attention)
from microserve_amd.kv_blocks import compact_kv_blocks, copy_kv_blocks  # noqa: F401
from microserve_amd.shared_prefix import (  # noqa: F401
    fp8_shared_prefix_decode_attention, group_by_prefix)
from microserve_amd.attention_weights import (  # noqa: F401
    allocate_attention_weights, clear_attention_weights, evict_kv_tokens,
    fp8_decode_attention_weights, fp8_window_attention_weights, select_kv_tokens)
from microserve_amd.attention import Attention  # noqa: F401
