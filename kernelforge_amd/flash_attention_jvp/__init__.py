"""FlashAttention forward/JVP drop-in (mirrors flash_attention_jvp/__init__.py:3-15)
plus the fused single-pass ``flash_attention_fwd_jvp``, the standalone backward
``flash_attention_backward``, and attention over a paged 8-bit key/value cache
(``paged_attention`` and the operators that keep the cache)."""

from .custom import (
    FlashAttentionFunction,
    flash_attention,
    flash_attention_backward,
    flash_attention_fwd_jvp,
    flash_attention_jvp,
    get_jvp_config,
)
from .paged import PagedKVCache, paged_attention, paged_block_tables_, paged_cache_append_, paged_kv_cache

__all__ = [
    "FlashAttentionFunction",
    "flash_attention",
    "flash_attention_backward",
    "flash_attention_jvp",
    "flash_attention_fwd_jvp",
    "get_jvp_config",
    "PagedKVCache",
    "paged_attention",
    "paged_block_tables_",
    "paged_cache_append_",
    "paged_kv_cache",
]
