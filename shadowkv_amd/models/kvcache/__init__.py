"""ShadowKV cache classes and the method registry (reference: models/kvcache/__init__.py:15-29).

Of the reference's policies only the ShadowKV offload class is provided: the others are not on
the sparse-decode path. "kv8" is the 8-bit full cache, which the reference does not have.
"""
from .base import KVCacheBase
from .kv8 import KV8Cache
from .shadow import ShadowKVCache_CPU

method2kvcache = {
    "shadowkv_cpu": ShadowKVCache_CPU,
    "kv8": KV8Cache,
}

__all__ = ["KV8Cache", "KVCacheBase", "ShadowKVCache_CPU", "method2kvcache"]
