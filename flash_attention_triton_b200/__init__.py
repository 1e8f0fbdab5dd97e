"""B200-native (sm_100a) causal FlashAttention-2 with the public surface of flash-attention-triton.

Exports the same four names as the reference package (``src/flash_attention_triton/__init__.py:13``)
plus the autograd function, and what the reference has no counterpart of: packed sequences with grouped heads, and the paged key-value cache.
"""

from .api import (
    FlashAttentionV2Function,
    KernelsConfigV2,
    flash_attention_v2,
    flash_attention_v2_custom,
    init_to_zero_v2,
)
from .packed import flash_attention_packed
from .paged import append_kv_cache, flash_attention_decode, rotary_tables
from .partition import shard_range, shard_slab

__version__ = "0.1.0"

__all__ = [
    "FlashAttentionV2Function",
    "KernelsConfigV2",
    "append_kv_cache",
    "flash_attention_decode",
    "flash_attention_packed",
    "flash_attention_v2",
    "flash_attention_v2_custom",
    "init_to_zero_v2",
    "rotary_tables",
    "shard_range",
    "shard_slab",
]
