"""Paged caches of one layer: latent rows and rope keys in pages that sequences take as they grow,
share when they fork and give back when they end.

Counterpart of the reference's [batch, max_len, dim] caches (racetrack/models/deepseek.py:735-736)
for sequences of different lengths: `PagedCaches` holds the tables and buffers of the ops.page_* calls
and hands them over. Everything lives on the device and no call reads back, so a decode step that
grows the caches can be captured in a CUDA graph; `check` is the one call that waits, and raises when
an entry of a list was refused.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import ops


class PagedCaches:
    """kv bf16 [n_pages, page_size, kv_lora] and pe bf16 [n_pages, page_size, rope] (and any `extra`
    buffers, {name: (row shape, dtype)}), block_table int32 [max_seqs, max_pages], seq_lens int32
    [max_seqs], refcount int32 [n_pages], status int32 [2]. page_size: a power of two from 16 on."""

    def __init__(self, shape, n_pages: int, page_size: int, max_seqs: int, max_pages: int, device, *,
                 extra: Optional[dict] = None):
        if page_size < 16 or page_size & (page_size - 1):
            raise RuntimeError("PagedCaches: page_size must be a power of two, 16 or more")
        if min(n_pages, max_seqs, max_pages) < 1:
            raise RuntimeError("PagedCaches: n_pages, max_seqs and max_pages must be positive")
        zeros = lambda *size, dtype=torch.int32: torch.zeros(*size, device=device, dtype=dtype)
        self.page_size = page_size
        self.kv = zeros(n_pages, page_size, shape.kv_lora, dtype=torch.bfloat16)
        self.pe = zeros(n_pages, page_size, shape.rope, dtype=torch.bfloat16)
        self.extra = {name: zeros(n_pages, page_size, *row, dtype=dtype) for name, (row, dtype) in (extra or {}).items()}
        self.block_table = torch.full((max_seqs, max_pages), -1, device=device, dtype=torch.int32)
        self.seq_lens, self.refcount, self.status = zeros(max_seqs), zeros(n_pages), zeros(2)

    @property
    def buffers(self) -> tuple:
        return (self.kv, self.pe, *self.extra.values())

    def extend(self, tokens: int, seqs: Optional[torch.Tensor] = None, *,
               offsets: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Room for new tokens; the slots their rows go to (ops.page_extend)."""
        return ops.page_extend(self.block_table, self.seq_lens, self.refcount, self.status, tokens, self.page_size,
                               seqs, offsets=offsets)

    def append(self, rows, seqs: Optional[torch.Tensor] = None, *, offsets: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Room for new tokens and their rows, one tensor for each of `buffers` (ops.page_append)."""
        return ops.page_append(self.buffers, rows, self.block_table, self.seq_lens, self.refcount, self.status, seqs,
                               offsets=offsets)

    def fork(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        """dst[i] becomes a copy of src[i] (ops.page_fork)."""
        ops.page_fork(self.buffers, self.block_table, self.seq_lens, self.refcount, self.status, src, dst)

    def free(self, seqs: torch.Tensor) -> None:
        """The sequences end and give their pages back (ops.page_free)."""
        ops.page_free(self.block_table, self.seq_lens, self.refcount, seqs)

    def compact(self) -> torch.Tensor:
        """Packs the pages in use to the front: int32 [2], their number and how many moved (ops.page_compact)."""
        return ops.page_compact(self.buffers, self.block_table, self.refcount)

    def check(self) -> None:
        """Waits for the device and raises if an entry was refused since the last check."""
        refused, lacking = self.status.tolist()
        if refused:
            self.status.zero_()
            raise RuntimeError(f"PagedCaches: {refused} entries were refused ({lacking} pages were lacking)")
