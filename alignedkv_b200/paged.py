"""A cache in pages for a batch of sequences with lengths of their own.

`PageTable` hands out pages of a pool to sequences and takes them back; `PagedLayer` is one layer's pool, driven by the operators of
`paged_ops`.  The layers of a model share one table: a sequence's positions lie in the same pages of every layer's pool.

The reference has no counterpart (one length for the batch, one tensor per layer: extension/k_cache_file.py:34-53).
"""
from __future__ import annotations

import torch

from . import paged_ops
from .extension._planes import cdiv

__all__ = ["PageTable", "PagedLayer", "FORMATS"]

FORMATS = ("fp16", "e4m3", "e2m1")


class PageTable:
    """Which pages hold the sequences' tokens.  pages int32 [B, width] and lens int32 [B] lie on the device, as the operators take them;
    `lengths` are the same numbers as lens on the host.

      table.reserve(n)        pages for n more tokens (a number, or one per sequence)
      layer.append(...)       ... of every layer, at positions lens ..
      table.advance(n)        they count from now on
      table.release(b)        sequence b is over, its pages are free; until tokens are reserved for it again, over[b] is true

    A page has one owner, and `pages` holds what was handed out: nothing else writes it.  (The operators take tables in which sequences share pages, or
    have given some up; such a table is the caller's own.)"""
    def __init__(self, bsz: int, max_seq_len: int, n_pages: int, page_size: int, device):
        if bsz < 1 or max_seq_len < 1 or n_pages < 1:
            raise ValueError(f"{bsz} sequences of up to {max_seq_len} tokens in {n_pages} pages")
        self.B, self.L, self.page_size, self.n_pages = bsz, max_seq_len, page_size, n_pages
        self.device = torch.device(device)
        self.width = cdiv(max_seq_len, page_size)
        self.pages = torch.full((bsz, self.width), -1, dtype=torch.int32, device=self.device)
        self.lens = torch.zeros(bsz, dtype=torch.int32, device=self.device)
        self.lengths = [0] * bsz
        self.owned = [[] for _ in range(bsz)]
        self.over = [False] * bsz
        self.free = list(range(n_pages - 1, -1, -1))

    def _counts(self, n) -> list:
        counts = [int(n)] * self.B if isinstance(n, int) else [int(x) for x in n]
        if len(counts) != self.B or min(counts) < 0:
            raise ValueError(f"expected a number of tokens for each of {self.B} sequences")
        return counts

    def reserve(self, n) -> None:
        """Pages for n more tokens of every sequence (a number or B of them); a refused call changes nothing."""
        counts = self._counts(n)
        need = []
        for b, c in enumerate(counts):
            if self.lengths[b] + c > self.L:
                raise RuntimeError(f"sequence {b}: no room for {c} tokens behind {self.lengths[b]} of {self.L}")
            need.append(max(0, cdiv(self.lengths[b] + c, self.page_size) - len(self.owned[b])))
        if sum(need) > len(self.free):
            raise RuntimeError(f"{sum(need)} pages are needed, {len(self.free)} of {self.n_pages} are free")
        places = []
        self.over = [o and not c for o, c in zip(self.over, counts)]
        for b, m in enumerate(need):
            for _ in range(m):
                page = self.free.pop()
                places.append((b, len(self.owned[b]), page))
                self.owned[b].append(page)
        if places:
            x = torch.tensor(places, device=self.device)
            self.pages[x[:, 0], x[:, 1]] = x[:, 2].to(torch.int32)

    def advance(self, n) -> None:
        """n tokens more of every sequence (a number or B of them) count as cached; their pages are reserved."""
        counts = self._counts(n)
        for b, c in enumerate(counts):
            if self.lengths[b] + c > len(self.owned[b]) * self.page_size:
                raise RuntimeError(f"sequence {b}: {c} tokens behind {self.lengths[b]} have no pages (reserve them first)")
        if len(set(counts)) == 1:
            self.lens += counts[0]
        else:
            self.lens += torch.tensor(counts, dtype=torch.int32, device=self.device)
        self.lengths = [a + c for a, c in zip(self.lengths, counts)]

    def release(self, b: int) -> None:
        """Sequence b has no tokens any more, its pages are free for others."""
        self.free.extend(reversed(self.owned[b]))
        self.owned[b] = []
        self.lengths[b] = 0
        self.over[b] = True
        self.pages[b] = -1
        self.lens[b] = 0


class PagedLayer:
    """One layer's pool of pages for keys and values of n_heads KV heads; form "fp16" (as they are), "e4m3" (8 bits and an exponent per token
    and head) or "e2m1" (4 bits, a scale per 16 channels, an exponent per token and head)."""
    def __init__(self, n_pages: int, page_size: int, n_heads: int, head_dim: int, device, form: str = "e4m3"):
        if form not in FORMATS:
            raise ValueError(f"form must be one of {FORMATS}")
        self.form, self.device = form, torch.device(device)
        shape = (n_pages, n_heads, page_size)
        row = head_dim // 2 if form == "e2m1" else head_dim
        dtype = {"fp16": torch.half, "e4m3": torch.float8_e4m3fn, "e2m1": torch.uint8}[form]
        make = lambda d, *more: torch.zeros(shape + more, dtype=d, device=self.device)  # noqa: E731
        self.k_codes, self.v_codes = make(dtype, row), make(dtype, row)
        self.k_exps, self.v_exps = (None, None) if form == "fp16" else (make(torch.int8), make(torch.int8))
        self.k_scales, self.v_scales = (make(torch.float8_e4m3fn, head_dim // 16), make(torch.float8_e4m3fn, head_dim // 16)) \
            if form == "e2m1" else (None, None)

    def append(self, k: torch.Tensor, v: torch.Tensor, table: PageTable, counts: torch.Tensor | None = None) -> None:
        """`paged_ops.paged_append` behind the table's tokens, whose pages are reserved; `table.advance` follows once for all layers."""
        paged_ops.paged_append(self, k, v, table.pages, table.lens, counts=counts)

    def read(self, table: PageTable, most: int, lens: torch.Tensor | None = None) -> tuple:
        """`paged_ops.paged_read`; lens: in the place of the table's."""
        return paged_ops.paged_read(self, table.pages, table.lens if lens is None else lens, most)

    def attention(self, q: torch.Tensor, table: PageTable, lens: torch.Tensor | None = None, **more):
        """`paged_ops.paged_attention`; lens: in the place of the table's."""
        return paged_ops.paged_attention(self, q, table.pages, table.lens if lens is None else lens, **more)
