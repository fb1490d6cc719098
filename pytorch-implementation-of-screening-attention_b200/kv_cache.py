"""Paged K/V cache for KV-cached generation.

Pages are [num_pages, H, page_size, D] tensors of UNIT key/value rows per
layer; a block table [B, max_blocks] maps each sequence's logical block to a
physical page.  Because the softmask is exactly zero beyond the window
(multiscreen/attention.py:117-118), no key older than t - (ceil(max w) - 1)
is ever read again, so each sequence only owns `pages_per_seq` pages used as
a ring: logical block lb lives in page b * pages_per_seq + lb % pages_per_seq.
With pages_per_seq >= ceil(keep / page_size) + 1 every block inside the
window maps to a distinct page, and the table never changes after set-up.

`quantize="int8"` keeps the rows as int8 with an fp32 scale each (68 bytes a row
for D = 64 instead of 128; see paged_append), half the bytes that a decode step
over long windows reads.  `max_draft` reserves ring rows for drafted tokens
behind the newest one (append_tree_decode, commit).
"""
from __future__ import annotations

import math

import torch

from . import _lib, paged


class PagedKVCache:
    def __init__(self, num_layers: int, batch: int, num_heads: int, head_dim: int, max_len: int,
                 max_window: float, dtype: torch.dtype, device: torch.device,
                 page_size: int = 64, quantize: str | None = None, max_draft: int = 0):
        if quantize not in (None, "int8"):
            raise ValueError(f"quantize is None or 'int8', got {quantize!r}")
        if max_draft < 0:
            raise ValueError("max_draft must not be negative")
        self.num_layers, self.batch = num_layers, batch
        self.num_heads, self.head_dim = num_heads, head_dim
        self.page_size = page_size
        self.quantize, self.max_draft = quantize, max_draft
        self.dtype = dtype            # of the rows given and returned
        self.max_window = max_window
        dmax = max(0, int(math.ceil(max_window)) - 1)
        # keys a decode step can still see: positions t - dmax .. t
        self.keep = min(max_len, dmax + 1)
        self.max_blocks = max(1, math.ceil((max_len + max_draft) / page_size))
        self.pages_per_seq = min(self.max_blocks,
                                 math.ceil((self.keep + max_draft) / page_size) + 1)
        num_pages = batch * self.pages_per_seq
        # every layer's pages in one allocation, so that a commit is one launch
        shape = (num_layers, num_pages, num_heads, page_size, head_dim)
        pdt = torch.int8 if quantize else dtype
        self._k_all = torch.zeros(shape, dtype=pdt, device=device)
        self._v_all = torch.zeros_like(self._k_all)
        self.k_pages, self.v_pages = list(self._k_all.unbind(0)), list(self._v_all.unbind(0))
        self._ks_all = self._vs_all = None
        self.k_scales = self.v_scales = [None] * num_layers
        if quantize:
            self._ks_all = torch.zeros(shape[:-1], dtype=torch.float32, device=device)
            self._vs_all = torch.zeros_like(self._ks_all)
            self.k_scales, self.v_scales = list(self._ks_all.unbind(0)), list(self._vs_all.unbind(0))
        lb = torch.arange(self.max_blocks, dtype=torch.int32)
        table = (torch.arange(batch, dtype=torch.int32).unsqueeze(1) * self.pages_per_seq
                 + (lb % self.pages_per_seq).unsqueeze(0))
        self.block_table = table.to(device)
        self._workspace = None
        self.num_splits = paged.decode_splits(batch * num_heads, self.keep, page_size)

    def nbytes(self) -> int:
        every = self.k_pages + self.v_pages + [t for t in self.k_scales + self.v_scales
                                               if t is not None]
        return sum(p.numel() * p.element_size() for p in every)

    def _pages(self, layer: int):
        return (self.k_pages[layer], self.v_pages[layer], self.block_table, self.k_scales[layer],
                self.v_scales[layer])

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
               eps: float = 1e-8) -> None:
        """Write unit rows of raw k, v (B,n,H,D) at positions[b] + (0..n-1)."""
        dt = self.dtype
        if self.quantize:
            paged.paged_append(k.to(dt), v.to(dt), positions, *self._pages(layer), eps=eps)
            return
        _lib.screen_kv_append(k.to(dt), v.to(dt), positions, self.k_pages[layer],
                              self.v_pages[layer], self.block_table, eps)

    def read(self, layer: int, positions: torch.Tensor, n: int):
        """(k, v) (B,n,H,D): the values of the cached rows at positions[b] +
        (0..n-1), in the cache's dtype."""
        return paged.paged_read(positions, n, *self._pages(layer), dtype=self.dtype)

    def append_decode(self, layer: int, k: torch.Tensor, v: torch.Tensor,
                      positions: torch.Tensor, q: torch.Tensor, seq_lens: torch.Tensor,
                      r: torch.Tensor, w: torch.Tensor, eps: float = 1e-8):
        """append(layer, k, v, positions) of one new row per sequence, then
        decode(layer, q, ...), in one launch.  An int8 cache takes the new row to
        be the newest (seq_lens = positions + 1) and returns None for |o|."""
        dt = self.dtype
        if self.quantize:
            if k.shape[1] != 1:
                raise ValueError("append_decode appends one row per sequence")
            y = paged.paged_tree_decode(q.to(dt).unsqueeze(1), k.to(dt), v.to(dt), positions, None,
                                        r, w, *self._pages(layer), max_window=self.max_window,
                                        eps=eps)
            return y.squeeze(1), None
        if self._workspace is None:
            need = self.batch * self.num_heads * self.num_splits * self.head_dim * 4
            self._workspace = torch.empty(need + 256, dtype=torch.uint8, device=q.device)
        return _lib.screen_decode_append(k.to(dt), v.to(dt), positions, q.to(dt), seq_lens, r, w,
                                         self.k_pages[layer], self.v_pages[layer],
                                         self.block_table, eps, self.num_splits, self._workspace)

    def decode(self, layer: int, q: torch.Tensor, seq_lens: torch.Tensor, r: torch.Tensor,
               w: torch.Tensor, eps: float = 1e-8):
        """Screening decode of raw q (B,H,D) for the newest token of each sequence:
        (y, |o|), |o| None for an int8 cache."""
        if self.quantize:
            return paged.paged_decode(q.to(self.dtype), seq_lens, r, w, *self._pages(layer),
                                      max_window=self.max_window, eps=eps), None
        if self._workspace is None:
            need = self.batch * self.num_heads * self.num_splits * self.head_dim * 4
            self._workspace = torch.empty(need + 256, dtype=torch.uint8, device=q.device)
        return _lib.screen_decode(q.to(self.dtype), seq_lens, r, w, self.k_pages[layer], self.v_pages[layer],
                                  self.block_table, eps, self.num_splits, self._workspace)

    def append_tree_decode(self, layer: int, k: torch.Tensor, v: torch.Tensor, q: torch.Tensor,
                           lens: torch.Tensor, parents: torch.Tensor | None, r: torch.Tensor,
                           w: torch.Tensor, eps: float = 1e-8) -> torch.Tensor:
        """The rows of a tree of n drafted tokens per sequence (raw q, k, v
        (B,n,H,D); see paged_tree_decode) written behind the lens[b] cached
        tokens, and the attention of every node: y (B,n,H,D).  n is at most
        max_draft + 1, the rows the ring has room for."""
        n = q.shape[1]
        if n > self.max_draft + 1:
            raise ValueError(f"a tree of {n} nodes in a cache made for max_draft={self.max_draft}")
        dt = self.dtype
        return paged.paged_tree_decode(q.to(dt), k.to(dt), v.to(dt), lens, parents, r, w,
                                       *self._pages(layer), max_window=self.max_window, eps=eps)

    def commit(self, lens: torch.Tensor, path: torch.Tensor, counts: torch.Tensor) -> None:
        """Keep the accepted path of a tree in every layer: row lens[b] + path[b,i]
        moves to lens[b] + i for i < counts[b] (see paged_commit)."""
        paged.paged_commit(lens, path, counts, self._k_all, self._v_all, self.block_table,
                           self._ks_all, self._vs_all)
