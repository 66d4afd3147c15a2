"""A full KV cache in 8 bits on the device, for layers that attend to everything (or to a sliding window and the
sequence's first tokens) rather than to a selection. No reference counterpart.

Keys and values are e4m3 codes [layers, B, H, max_length, 128] with one float32 power of two per block of
`block` tokens and head (shadowkv.kv8_write, kv8_attn, kv8_read): half the bytes of bf16, quantised as they are
written. The lengths live on the device and the step advances them itself, at layer 0, so prompts of different
lengths share a batch and a captured step stays valid as the cache grows.
"""
from __future__ import annotations

import torch

from ...kernels import shadowkv
from .base import KVCacheBase


class KV8Cache(KVCacheBase):
    """Every layer's keys and values in 8 bits; a step updates the layers in order, from layer 0."""

    def __init__(self, config, batch_size: int = 1, max_length: int = 32 * 1024, device: str = "cuda:0",
                 dtype=torch.bfloat16, block: int = 64, window: int | None = None, sinks: int = 0) -> None:
        self.config = config
        self.batch_size = batch_size
        self.max_length = max_length
        self.device = device
        self.dtype = dtype
        self.num_key_value_groups = config.num_attention_heads // config.num_key_value_heads
        self.head_dim = config.hidden_size // config.num_attention_heads
        self.num_attention_heads = config.num_attention_heads
        self.num_key_value_heads = config.num_key_value_heads
        self.num_layers = config.num_hidden_layers
        if self.head_dim != 128 or dtype != torch.bfloat16:
            raise ValueError(f"KV8Cache takes bf16 heads of 128 dims, not {dtype} of {self.head_dim}")
        if block not in shadowkv.KV8_BLOCKS:
            raise ValueError(f"block={block} must be one of {shadowkv.KV8_BLOCKS}")
        if not 1 <= max_length <= shadowkv.KV8_MAX_TOKENS:
            raise ValueError(f"max_length={max_length} must be 1 to {shadowkv.KV8_MAX_TOKENS}")
        if (window is not None and not 1 <= window < 2 ** 31) or not 0 <= sinks < 2 ** 31 or (sinks and window is None):
            raise ValueError(f"window={window} sinks={sinks} (a window of at least 1; sinks need one)")
        self.block, self.window, self.sinks = block, window, sinks

        shape = (self.num_layers, batch_size, self.num_key_value_heads, max_length, self.head_dim)
        blocks = (max_length + block - 1) // block
        # What no sequence holds is never used, so the codes need no clearing, here or in clear().
        self.k8, self.v8 = (torch.empty(shape, dtype=torch.float8_e4m3fn, device=device) for _ in range(2))
        self.k_scale, self.v_scale = (torch.empty(*shape[:3], blocks, dtype=torch.float32, device=device)
                                      for _ in range(2))
        self.lengths = torch.zeros(batch_size, dtype=torch.int32, device=device)  # tokens held, new ones among them
        self.start = torch.zeros(batch_size, dtype=torch.int32, device=device)  # where this step's tokens begin
        self.counts = None  # this step's tokens of each sequence, or None: all that were given
        self.incoming = 0
        self.kv_offset = 0  # the host's bound on the longest sequence: padded rows count (until trim())
        self.unfinished = 0  # tokens of a step that has not reached the last layer: held, and not in kv_offset yet

    def print_stats(self):
        seen = "all" if self.window is None else f"{self.window} + {self.sinks}"
        print(f"KV8 | block {self.block} | seen {seen} | cached {self.kv_offset} of {self.max_length}")

    def check_capacity(self, incoming: int = 1):
        if self.kv_offset + self.unfinished + incoming > self.max_length:
            raise RuntimeError(f"cache capacity exhausted: {self.kv_offset + self.unfinished} of {self.max_length} tokens "
                               f"held, {incoming} new; construct the cache with a larger max_length")

    def advance(self, incoming: int = 1):
        """Host bookkeeping of one step (the device lengths advance inside the step): a replayed one, or one that is
        complete without this cache's last layer."""
        self.kv_offset += incoming
        if incoming == self.unfinished:
            self.unfinished = 0

    def update_kv_cache(self, new_k_cache: torch.Tensor, new_v_cache: torch.Tensor, layer_idx: int,
                        counts: torch.Tensor | None = None):
        """Append the new tokens [B, H, T, 128] of one layer: the first counts[b] rows of each sequence (device int32
        [B]; all T without it). Layer 0's counts are the whole step's: the other layers may be given them too, and
        theirs are not read."""
        incoming = new_k_cache.shape[-2]
        if layer_idx == 0:
            self.check_capacity(incoming)
            self.start.copy_(self.lengths)
        elif incoming != self.incoming:
            raise ValueError(f"layer {layer_idx} got {incoming} tokens in a step of {self.incoming}")
        elif counts is not None and self.counts is None:
            raise ValueError(f"layer {layer_idx} got counts in a step whose layer 0 had none")
        shadowkv.kv8_write(new_k_cache, new_v_cache, self.k8[layer_idx], self.v8[layer_idx], self.k_scale[layer_idx],
                           self.v_scale[layer_idx], self.start, counts if layer_idx == 0 else self.counts,
                           block=self.block)
        if layer_idx == 0:  # (behind the write: one that is refused leaves the lengths)
            self.lengths.add_(incoming if counts is None else counts.clamp(0, incoming))
            if self.unfinished:  # a step that ended before the last layer: its tokens are held
                self.advance(self.unfinished)
            self.counts, self.incoming, self.unfinished = counts, incoming, incoming
        if layer_idx == self.num_layers - 1:
            self.advance(self.unfinished)

    def trim(self, lengths: torch.Tensor, longest: int):
        """Between steps: keep the first min(lengths[b], longest) tokens of each sequence (lengths: device int32 [B]; all
        that it holds if those are fewer) and drop the others: drafted ones that were rejected, or a step that failed on
        its way. The capacity is counted from `longest` on: cache.lengths with the longest sequence's tokens takes the
        padding of a ragged batch out of it. A captured trim() takes max_length, and kv_offset is set beside its
        replays."""
        if lengths.dtype != torch.int32 or lengths.shape != self.lengths.shape or lengths.device != self.lengths.device:
            raise ValueError(f"lengths must be {self.batch_size} int32 on {self.lengths.device}, got "
                             f"{tuple(lengths.shape)} {lengths.dtype} on {lengths.device}")
        if longest < 0:
            raise ValueError(f"longest={longest} must not be negative")
        self.lengths.copy_(torch.minimum(self.lengths, lengths.clamp(0, longest)))
        self.kv_offset = min(self.kv_offset + self.unfinished, longest)
        self.unfinished = self.incoming = 0
        self.counts = None

    def attend(self, query_states: torch.Tensor, layer_idx: int) -> torch.Tensor:
        """Attention of this step's queries [B, Hq, T, 128] over the layer, their own keys in it -> [B, T, Hq, 128];
        zeros past counts[b]."""
        if query_states.shape[-2] != self.incoming:
            raise ValueError(f"{query_states.shape[-2]} queries in a step of {self.incoming} tokens")
        return shadowkv.kv8_attn(query_states, self.k8[layer_idx], self.v8[layer_idx], self.k_scale[layer_idx],
                                 self.v_scale[layer_idx], self.lengths, self.counts, block=self.block,
                                 window=self.window, sinks=self.sinks)

    def get_kv(self, layer_idx: int, start: int, rows: int):
        """Rows [start, start + rows) of every sequence of the layer as bf16 keys and values [B, H, rows, 128] (what
        was written, rounded to the cache's codes; rows behind a sequence's last are arbitrary)."""
        return (shadowkv.kv8_read(self.k8[layer_idx], self.k_scale[layer_idx], start, rows, block=self.block),
                shadowkv.kv8_read(self.v8[layer_idx], self.v_scale[layer_idx], start, rows, block=self.block))

    def H2D(self):
        torch.cuda.synchronize(self.device)  # all of it is on the device already

    def clear(self):
        self.lengths.zero_()
        self.start.zero_()
        self.counts = None
        self.incoming = 0
        self.kv_offset = 0
        self.unfinished = 0

    def get_kv_len(self):
        return self.kv_offset
