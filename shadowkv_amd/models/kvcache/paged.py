"""A full KV cache in pages that sequences of different lengths share, for serving: a sequence takes pages as it grows and
gives them back when it ends, so memory goes by the tokens that are held rather than by batch_size * max_length. No
reference counterpart.

Keys and values are bf16 [layers, pages, H, page, 128] (shadowkv.paged_write, paged_attn). Lengths, tables and the free
pages live on the device, where a step takes what it needs at layer 0 (shadowkv.paged_reserve): nothing is asked of the
host, and a captured step stays valid as sequences grow, end and begin.
"""
from __future__ import annotations

import torch

from ...kernels import shadowkv
from .base import KVCacheBase


class PagedKVCache(KVCacheBase):
    """Every layer's keys and values in pages; a step updates the layers in order, from layer 0. Sequence b of batch_size
    is a place that one sequence after the other may take."""

    def __init__(self, config, batch_size: int = 1, max_length: int = 32 * 1024, device: str = "cuda:0",
                 dtype=torch.bfloat16, page: int = 64, pages: int | None = None, window: int | None = None) -> None:
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
            raise ValueError(f"PagedKVCache takes bf16 heads of 128 dims, not {dtype} of {self.head_dim}")
        if page not in shadowkv.PAGE_SIZES:
            raise ValueError(f"page={page} must be one of {shadowkv.PAGE_SIZES}")
        width = -(-max_length // page)
        if max_length < 1 or width * page > shadowkv.PAGED_MAX_TOKENS:
            raise ValueError(f"max_length={max_length} must be 1 to {shadowkv.PAGED_MAX_TOKENS}")
        pages = batch_size * width if pages is None else pages
        if not 1 <= pages <= 2 ** 31 // page:
            raise ValueError(f"pages={pages} must be 1 to 2^31 tokens")
        if window is not None and not 1 <= window < 2 ** 31:
            raise ValueError(f"window={window} must be at least 1")
        self.page, self.pages, self.window = page, pages, window

        # What no sequence holds is never used, so the pages need no clearing, here or in clear().
        shape = (self.num_layers, pages, self.num_key_value_heads, page, self.head_dim)
        self.k_pages, self.v_pages = (torch.empty(shape, dtype=dtype, device=device) for _ in range(2))
        ints = lambda *n: torch.zeros(n, dtype=torch.int32, device=device)  # noqa: E731
        self.table = ints(batch_size, width).fill_(-1)
        self.held, self.free_pages, self.free_count = ints(batch_size), ints(pages), ints(1)
        self.lengths, self.start = ints(batch_size), ints(batch_size)  # tokens held; where the last step's begin
        self.asked = ints(batch_size)  # new tokens of each sequence in that step
        self.unserved = torch.zeros(batch_size, dtype=torch.bool, device=device)  # which it left as they were
        # Of that step: its rows' places, the sequences' tokens (0: not served), where the rows are stored.
        self.cu, self.totals, self.slots = ints(batch_size + 1), ints(batch_size), ints(0)
        self.incoming = 0  # its rows
        self.max_new = 1   # the host's bound on a sequence's new tokens
        self.kv_offset = 0  # the host's bound on the longest sequence
        self.unfinished = 0  # tokens of a step that has not reached the last layer: held, and not in kv_offset yet
        self.clear()

    def print_stats(self):
        seen = "all" if self.window is None else f"{self.window}"
        print(f"Paged KV | {self.pages} pages of {self.page} | seen {seen} | longest {self.kv_offset} of {self.max_length}")

    def check_capacity(self, incoming: int = 1):
        """That no sequence passes max_length. Whether there are pages is known on the device alone: refused()."""
        if self.kv_offset + self.unfinished + incoming > self.max_length:
            raise RuntimeError(f"cache capacity exhausted: {self.kv_offset + self.unfinished} of {self.max_length} tokens "
                               f"held, {incoming} new; construct the cache with a larger max_length")

    def advance(self, incoming: int = 1):
        """Host bookkeeping of one step (the device lengths advance inside the step): a replayed one, or one that is
        complete without this cache's last layer."""
        self.kv_offset += incoming
        if incoming == self.unfinished:
            self.unfinished = 0

    def _packed(self, x: torch.Tensor) -> torch.Tensor:
        """[B, heads, T, 128] (of packed rows: B = 1) as rows [B * T, heads, 128]."""
        return x.transpose(1, 2).flatten(0, 1)

    def update_kv_cache(self, new_k_cache: torch.Tensor, new_v_cache: torch.Tensor, layer_idx: int,
                        counts: torch.Tensor | None = None, max_new: int | None = None):
        """Append the new tokens of one layer: T of each sequence, [batch_size, H, T, 128], or with counts (device int32
        [batch_size]) packed rows [1, H, N, 128], counts[b] of sequence b behind those of the sequences before it; rows
        behind the last are padding. max_new: the host's bound on counts (default: N), by which the capacity is counted. A
        sequence that lacks pages, or has more new tokens than max_new, is left as it is (refused()). Layer 0's counts are
        the whole step's: the other layers may be given them too, and theirs are not read."""
        k, v = self._packed(new_k_cache), self._packed(new_v_cache)
        rows = k.shape[0]
        if layer_idx == 0:
            if new_k_cache.shape[0] != (self.batch_size if counts is None else 1):
                raise ValueError(f"keys {tuple(new_k_cache.shape)} must be [{self.batch_size}, H, T, 128], or with counts "
                                 "[1, H, N, 128]")
            if max_new is not None and max_new < 1:
                raise ValueError(f"max_new={max_new}")
            new = new_k_cache.shape[2] if counts is None or max_new is None else min(max_new, rows)
            self.check_capacity(new)
            if counts is None:
                self.asked.fill_(new)
            else:
                if counts.shape != self.asked.shape or counts.dtype != torch.int32:
                    raise ValueError(f"counts must be {self.batch_size} int32, got {tuple(counts.shape)} {counts.dtype}")
                self.asked.copy_(counts)
            self.start.copy_(self.lengths)
            # (one with more new tokens than the bound is left as it is: no length is the reserve's sign for that; one
            # with more than there are rows is by itself)
            lengths = self.lengths
            if counts is not None and new < rows:
                lengths = lengths.masked_fill(self.asked > new, -1)
            self.cu, self.totals, self.slots = shadowkv.paged_reserve(
                lengths, self.asked, self.table, self.held, self.free_pages, self.free_count, rows=rows, page=self.page)
            # (here, where a replay's go too: a captured step's totals are its graph's own)
            torch.eq(self.totals, 0, out=self.unserved)
        elif rows != self.incoming:
            raise ValueError(f"layer {layer_idx} got {rows} rows in a step of {self.incoming}")
        shadowkv.paged_write(k, v, self.k_pages[layer_idx], self.v_pages[layer_idx], self.slots)
        if layer_idx == 0:  # (behind the write: one that is refused leaves the lengths)
            torch.maximum(self.lengths, self.totals, out=self.lengths)
            if self.unfinished:  # a step that ended before the last layer: its tokens are held
                self.advance(self.unfinished)
            self.incoming, self.max_new, self.unfinished = rows, max(new, 1), new
        if layer_idx == self.num_layers - 1:
            self.advance(self.unfinished)

    def refused(self) -> torch.Tensor:
        """Which sequences' tokens the last step (an eager or a replayed one) did not take (device bool [batch_size]), for
        lack of pages or as more than its max_new: their outputs are zeros. They can be given again, when others have ended
        or in pieces."""
        return self.unserved & (self.asked > 0)

    def trim(self, lengths: torch.Tensor, longest: int):
        """Between steps: keep the first min(lengths[b], longest) tokens of each sequence (lengths: device int32
        [batch_size]; all that it holds if those are fewer) and give the pages behind them back: rejected drafts, a step
        that failed on its way, and with 0 a sequence that has ended, whose place another one may take. The capacity is
        counted from `longest` on. A captured trim() takes max_length, and kv_offset is set beside its replays."""
        if lengths.dtype != torch.int32 or lengths.shape != self.lengths.shape or lengths.device != self.lengths.device:
            raise ValueError(f"lengths must be {self.batch_size} int32 on {self.lengths.device}, got "
                             f"{tuple(lengths.shape)} {lengths.dtype} on {lengths.device}")
        if longest < 0:
            raise ValueError(f"longest={longest} must not be negative")
        shadowkv.paged_release(self.lengths, lengths.clamp(0, longest), self.table, self.held, self.free_pages,
                               self.free_count, page=self.page)
        self.kv_offset = min(self.kv_offset + self.unfinished, longest)
        self.unfinished = self.incoming = 0

    def attend(self, query_states: torch.Tensor, layer_idx: int) -> torch.Tensor:
        """Attention of this step's queries, [B, Hq, T, 128] as the keys were given, over the layer, their own keys in it
        -> [B, T, Hq, 128]; zeros for padding and for sequences that were refused."""
        q = self._packed(query_states)
        if q.shape[0] != self.incoming:
            raise ValueError(f"{q.shape[0]} queries in a step of {self.incoming} rows")
        out = shadowkv.paged_attn(q, self.k_pages[layer_idx], self.v_pages[layer_idx], self.table, self.totals, self.cu,
                                  max_new=self.max_new, window=self.window)
        return out.view(query_states.shape[0], query_states.shape[2], *out.shape[1:])

    def get_kv(self, layer_idx: int, sequence: int, rows: int):
        """The first `rows` keys and values of one sequence of the layer, [H, rows, 128] (those behind its last token are
        arbitrary)."""
        ids = self.table[sequence, :-(-rows // self.page)].long().clamp(min=0)
        return tuple(x[layer_idx][ids].transpose(0, 1).flatten(1, 2)[:, :rows] for x in (self.k_pages, self.v_pages))

    def H2D(self):
        torch.cuda.synchronize(self.device)  # all of it is on the device already

    def clear(self):
        self.lengths.zero_()
        self.start.zero_()
        self.asked.zero_()
        self.table.fill_(-1)
        self.held.zero_()
        self.free_pages.copy_(torch.arange(self.pages - 1, -1, -1, dtype=torch.int32, device=self.device))
        self.free_count.fill_(self.pages)
        self.incoming = 0
        self.kv_offset = 0
        self.unfinished = 0

    def get_kv_len(self):
        return self.kv_offset
