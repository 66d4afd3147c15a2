"""Cache-class -> attention-handler map (reference: models/attention/__init__.py:19-31)."""
from typing import Dict

from ..kvcache import KV8Cache, KVCacheBase, ShadowKVCache_CPU
from .base import AttentionBase
from .kv8 import KV8Attention
from .shadow import ShadowAttention

Cache2Attn: Dict[type, type] = {
    ShadowKVCache_CPU: ShadowAttention,
    KV8Cache: KV8Attention,
}

__all__ = ["AttentionBase", "KV8Attention", "ShadowAttention", "Cache2Attn", "KVCacheBase"]
