"""Attention handler of the 8-bit KV cache: RoPE, append, attention over what the cache holds. No reference
counterpart. Prompts, pieces of prompts, drafted tokens and single tokens take the same three steps, so a
query reads its own tokens as the cache holds them, whichever way they came."""
from __future__ import annotations

from .base import AttentionBase


class KV8Attention(AttentionBase):

    def prefill(self, query_states, key_states, value_states, position_ids, layer_idx, counts=None):
        """A prompt or the next piece of one, [B, Hq or H, T, 128] -> [B, T, Hq, 128]. counts (device int32 [B]): how
        many of the T rows each sequence has; the others are padding, stored nowhere and zeros in the result."""
        query_states, key_states = self.apply_rotary_pos_emb(query_states, key_states, position_ids)
        self.kv_cache.update_kv_cache(key_states, value_states, layer_idx, counts)
        return self.kv_cache.attend(query_states, layer_idx)

    def decode(self, query_states, key_states, value_states, position_ids, layer_idx, counts=None):
        """One new token of each sequence, or several drafted ones, through the layer."""
        return self.prefill(query_states, key_states, value_states, position_ids, layer_idx, counts)
