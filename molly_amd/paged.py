"""The paged key / value cache of a decoder: page pools for every layer and the pages each sequence owns (molly_hip.h: molly_paged_kv_*,
molly_attn_paged).  The reference's `generate` keeps HF's DynamicCache (reference: src/model/omics_one.py:220-232): a dense rectangle of the longest
padded prompt for every row; here a row holds the pages its own tokens need, in bf16 or in half the bytes as e4m3."""
from __future__ import annotations

from typing import List

import torch

from . import ops

BF16 = torch.bfloat16


class PagedKVCache:
    """Pools [layers, pages, kv heads, page size, dim] for K and V; dtype 'bf16' or 'e4m3' (with exponent bytes [layers, pages, kv heads, page size])."""

    def __init__(self, n_layers: int, n_pages: int, n_kv_heads: int, head_dim: int, page_size: int = 64, dtype: str = "bf16", device="cuda"):
        if dtype not in ("bf16", "e4m3"):
            raise ValueError(f"PagedKVCache: dtype must be 'bf16' or 'e4m3', got {dtype!r}")
        if head_dim not in (64, 128):
            raise ValueError(f"PagedKVCache: head_dim {head_dim} (built for 64 and 128)")
        if page_size not in (16, 32, 64, 128, 256):
            raise ValueError(f"PagedKVCache: page_size {page_size} (a power of two in 16..256)")
        if n_pages <= 0 or n_pages * page_size > 0x7fffffff:
            raise ValueError(f"PagedKVCache: {n_pages} pages of {page_size} places (1 .. 2^31 - 1 places)")
        self.page_size, self.n_pages, self.dtype = page_size, n_pages, dtype
        shape = (n_layers, n_pages, n_kv_heads, page_size, head_dim)
        self.kscale = self.vscale = None
        if dtype == "e4m3":
            self.k, self.v = (torch.empty(shape, dtype=torch.uint8, device=device).view(ops.E4M3) for _ in range(2))
            self.kscale, self.vscale = (torch.empty(shape[:4], dtype=torch.uint8, device=device) for _ in range(2))
        else:
            self.k, self.v = (torch.empty(shape, dtype=BF16, device=device) for _ in range(2))
        self._free = list(range(n_pages - 1, -1, -1))
        self._layers = [dict(kpool=self.k[i], vpool=self.v[i], kscale=None if self.kscale is None else self.kscale[i],
                             vscale=None if self.vscale is None else self.vscale[i]) for i in range(n_layers)]

    def layer(self, i: int) -> dict:
        """the pools of layer i, as the ops take them"""
        return self._layers[i]

    def pages_for(self, n_tokens: int) -> int:
        return -(-n_tokens // self.page_size)

    def allocate(self, n_tokens: int) -> List[int]:
        """Pages for a sequence of up to n_tokens; raises when the pool has too few."""
        n = self.pages_for(n_tokens)
        if n > len(self._free):
            raise RuntimeError(f"PagedKVCache: {n} pages wanted, {len(self._free)} of {self.n_pages} free")
        return [self._free.pop() for _ in range(n)]

    def free(self, pages: List[int]):
        """Give a sequence's pages back."""
        taken = set(self._free)
        for p in pages:
            if not 0 <= p < self.n_pages or p in taken:
                raise ValueError(f"PagedKVCache: page {p} is not allocated")
            taken.add(p)
        self._free += list(pages)

    def block_table(self, pages: List[List[int]]) -> torch.Tensor:
        """int32 [sequences, most pages], -1 behind a sequence's last page"""
        t = torch.full((len(pages), max([len(p) for p in pages] + [1])), -1, dtype=torch.int32)
        for b, p in enumerate(pages):
            t[b, :len(p)] = torch.tensor(p, dtype=torch.int32)
        return t.to(self.k.device)

    def copy_pages(self, src: torch.Tensor, dst: torch.Tensor):
        """Page dst[i] becomes a copy of page src[i] in every layer (all of src are read before any of dst is written)."""
        for i in range(self.k.shape[0]):
            for t in (self.k, self.v, self.kscale, self.vscale):
                if t is not None:
                    x = t[i].view(torch.uint8) if t.dtype == ops.E4M3 else t[i]
                    x[dst] = x[src]
