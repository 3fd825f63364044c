"""Device-resident KV caches for the attention path.

The reference keeps, per layer, a (k, v) pair of [B, Hkv, T_cached, D] tensors
that every step grows with torch.cat and then expands with repeat_interleave
(smollm.py:68-77, 198-208); its NPU decode route pads Tk to a bucket
(smollm.py:17-20, 144). Here the cache is allocated once at its maximum length
and written in place by npu_b200.api.rope_append, and the prefill/decode
kernels read it directly with per-sequence positions, GQA heads unexpanded.

Positions live on the device in two int32 vectors, so a step needs no host
synchronisation: every layer's append reads the step's start positions from
one and writes start + T into the other (the same value from each layer), the
attention reads lengths from the second, and `advance` copies the second into
the first on the device. The buffers never move, so a step can be captured in
a CUDA graph and replayed.

PagedKVCache keeps sequences of different lengths in pages of one pool instead
(npu_b200.api.rope_append_paged, prefill_varlen and decode_paged).
"""
from __future__ import annotations

import torch


class KVCache:
    """k, v: [n_layers, B, Hkv, max_len, head_dim] bf16 on `device`."""

    def __init__(self, n_layers: int, batch: int, n_kv_heads: int, max_len: int, head_dim: int,
                 device: torch.device):
        if min(n_layers, batch, n_kv_heads, max_len, head_dim) <= 0:
            raise ValueError("KVCache dimensions must be positive")
        shape = (n_layers, batch, n_kv_heads, max_len, head_dim)
        self.k = torch.zeros(shape, dtype=torch.bfloat16, device=device)
        self.v = torch.zeros(shape, dtype=torch.bfloat16, device=device)
        self._pos = torch.zeros((2, batch), dtype=torch.int32, device=device)
        self.max_len = max_len
        self.batch = batch

    @property
    def start(self) -> torch.Tensor:
        """int32 [B]: position of each sequence's next token (device)."""
        return self._pos[0]

    @property
    def end(self) -> torch.Tensor:
        """int32 [B]: positions after the step in progress (what the appends
        write and the attention reads as sequence lengths)."""
        return self._pos[1]

    def layer(self, i: int):
        return self.k[i], self.v[i]

    def advance(self) -> None:
        """Finish a step: the lengths written by this step become the next
        start (a device copy on the current stream)."""
        self._pos[0].copy_(self._pos[1])

    def reset(self, lengths=None) -> None:
        """Empty the cache (or set per-sequence lengths, e.g. after a prefill
        computed elsewhere); the stored K/V rows are left as they are."""
        if lengths is None:
            self._pos.zero_()
        else:
            self._pos[0].copy_(torch.as_tensor(lengths, dtype=torch.int32))
            self._pos[1].copy_(self._pos[0])

    def lengths(self) -> list:
        """Host copy of the current lengths (synchronises)."""
        return [int(x) for x in self.start.tolist()]


class PagedKVCache:
    """Page pools for sequences of different lengths: k, v [n_layers, n_pages,
    Hkv, page, head_dim] bf16 on `device`. Sequences take pages as they need
    them and give them back (`reserve`, `PagedSequences.release`), so the memory
    held follows the tokens stored instead of batch x longest. The pools are
    allocated once and never cleared: a page's old contents are not read.
    """

    def __init__(self, n_layers: int, n_pages: int, n_kv_heads: int, page: int, head_dim: int,
                 device: torch.device):
        if min(n_layers, n_pages, n_kv_heads, page, head_dim) <= 0:
            raise ValueError("PagedKVCache dimensions must be positive")
        if page % 16:
            raise ValueError(f"page must be a multiple of 16 tokens, got {page}")
        shape = (n_layers, n_pages, n_kv_heads, page, head_dim)
        self.k = torch.empty(shape, dtype=torch.bfloat16, device=device)
        self.v = torch.empty(shape, dtype=torch.bfloat16, device=device)
        self.page = page
        self.device = self.k.device
        self._free = list(range(n_pages - 1, -1, -1))

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def layer(self, i: int):
        return self.k[i], self.v[i]

    def reserve(self, capacities) -> "PagedSequences":
        """Pages for len(capacities) new, empty sequences of at most that many tokens each."""
        capacities = [int(c) for c in capacities]
        if not capacities or min(capacities) < 1:
            raise ValueError("capacities must be one or more positive token counts")
        counts = [-(-c // self.page) for c in capacities]
        if sum(counts) > len(self._free):
            raise ValueError(f"{sum(counts)} pages are needed and {len(self._free)} are free")
        return PagedSequences(self, [[self._free.pop() for _ in range(n)] for n in counts])


class PagedSequences:
    """A batch of sequences in a PagedKVCache: their block table and, like
    KVCache, two vectors of positions on the device, so that steps need no host
    synchronisation. `start`: the next token's position; `end`: the lengths
    after the step in progress; `advance` finishes a step."""

    def __init__(self, cache: PagedKVCache, pages: list):
        self.cache, self._pages = cache, pages
        self.batch = len(pages)
        # -1 is no page: a token past a sequence's own pages is left out and reported.
        table = torch.full((self.batch, max(len(p) for p in pages)), -1, dtype=torch.int32)
        for b, p in enumerate(pages):
            table[b, :len(p)] = torch.tensor(p, dtype=torch.int32)
        self.block_table = table.to(cache.device)
        self._pos = torch.zeros((2, self.batch), dtype=torch.int32, device=cache.device)
        # Offsets of a step of one token per sequence.
        self.one_each = torch.arange(self.batch + 1, dtype=torch.int32, device=cache.device)

    @property
    def start(self) -> torch.Tensor:
        return self._pos[0]

    @property
    def end(self) -> torch.Tensor:
        return self._pos[1]

    @property
    def released(self) -> bool:
        """Whether the pages are given back; block_table then names pages of others."""
        return not self._pages

    def advance(self) -> None:
        self._pos[0].copy_(self._pos[1])

    def lengths(self) -> list:
        """Host copy of the current lengths (synchronises)."""
        return [int(x) for x in self.start.tolist()]

    def release(self) -> None:
        """Give the pages back. Work already queued on the current stream may
        still read them; later owners are to use the same stream."""
        for p in self._pages:
            self.cache._free.extend(reversed(p))
        self._pages = []
