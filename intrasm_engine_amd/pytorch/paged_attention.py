"""A paged cache of keys and values for generation: tokens appended to it, single new tokens attending to it, pages selected.

Three operators under ``torch.ops.iex_ops`` (``csrc/host/paged_ops.h``), on the current stream, capturable, without a gradient:

    kv_append_(k, v, keys, values, page_table, lengths, offsets=None, q=None, rotation=None, interleaved=False, bounds=None,
               key_exponents=None, value_exponents=None) -> q, rotated (None without q)
    paged_attention(q, keys, values, page_table, lengths, scale=None, pages=None, key_exponents=None, value_exponents=None)
    select_pages(q, bounds, page_table, lengths, page_size, count, first=1, last=1) -> (sequences, kv_heads, count) int32

Tokens are (tokens, heads, head_dim) tensors of fp16 or bf16 with any strides; what comes back has the strides of ``q``, so the
(heads * head_dim, tokens) matrices that projections ``W @ X`` leave and take go in as ``x.view(heads, head_dim, tokens).permute(2, 0,
1)`` and come out the same way.  ``page_table``: (sequences, width) int32, the pages of every sequence in order; ``lengths``:
(sequences) int32, tokens of every sequence, the new ones of an append counted.  Both are read on the device when the kernels
run: a captured graph follows what they hold at each replay.  A length is cut to what the table holds; a page outside
the cache (-1, say) counts as given back: nothing is written to it, nothing of it is attended to, it is not selected.

:class:`KVCache` holds a cache's tensors and calls the three.
"""
from __future__ import annotations

import torch

ops = torch.ops.iex_ops


def rotation_table(positions: int, features: int, base: float = 10000.0, device=None) -> torch.Tensor:
    """(positions, features) float32 for ``kv_append_``: cosines, then sines, of position * base^(-2 j / features), j < features / 2;
    the angles in 64 bits (in 32, those of position 100000 are off by up to 0.004)."""
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * base ** (-2.0 * torch.arange(features // 2, dtype=torch.float64) / features)
    return torch.cat([angle.cos(), angle.sin()], 1).to(device=device, dtype=torch.float32)


class KVCache:
    """``pages`` pages of ``page_size`` (16 .. 256, a power of two) tokens for ``kv_heads`` heads of ``head_dim`` (64, 128 or 256).

    ``eight_bits``: e4m3 codes and, per token and head, the least power of two as their scale that brings the largest magnitude to
    448 (one byte; infinities become NaN and do not count), in place of ``dtype``: half the memory, and half the time of reading it.  ``bounds``: also keep the smallest and
    largest key of every page, head and feature, which :meth:`select` reads (they begin anew with a page's first token; tokens that are
    taken back, by a shorter length, and written again widen them at most).  Who has which page is the caller's business: two
    sequences may share pages that neither appends to (a common prefix)."""

    def __init__(self, pages: int, page_size: int, kv_heads: int, head_dim: int, dtype=torch.float16, device="cuda", eight_bits: bool = False,
                 bounds: bool = False):
        self.page_size, self.kv_heads, self.head_dim, self.dtype = page_size, kv_heads, head_dim, dtype
        stored = torch.float8_e4m3fn if eight_bits else dtype
        self.keys = torch.empty(pages, kv_heads, page_size, head_dim, dtype=stored, device=device)
        self.values = torch.empty_like(self.keys)
        self.key_exponents = self.value_exponents = self.bounds = None
        if eight_bits:
            self.key_exponents = torch.empty(pages, kv_heads, page_size, dtype=torch.uint8, device=device)
            self.value_exponents = torch.empty_like(self.key_exponents)
        if bounds:
            self.bounds = torch.empty(pages, kv_heads, 2, head_dim, dtype=dtype, device=device)

    def append_(self, k, v, page_table, lengths, offsets=None, q=None, rotation=None, interleaved: bool = False):
        """Write the newest tokens' keys and values, (tokens, kv_heads, head_dim): token s is sequence s's, or ``offsets[s] ..
        offsets[s + 1]`` are (int32, from 0).  Keys and ``q`` are rotated by ``rotation`` (:func:`rotation_table`; a row for every
        position that the table can hold) at their positions.  Returns q so."""
        return ops.kv_append_(k, v, self.keys, self.values, page_table, lengths, offsets, q, rotation, interleaved, self.bounds, self.key_exponents,
                              self.value_exponents)

    def attend(self, q, page_table, lengths, scale: float | None = None, pages=None):
        """softmax(scale q k^T) v over each sequence's tokens, or those of its listed ``pages`` (:meth:`select`); q: (sequences, heads,
        head_dim), heads a multiple of ``kv_heads``; ``scale``: 1 / sqrt(head_dim)."""
        return ops.paged_attention(q, self.keys, self.values, page_table, lengths, scale, pages, self.key_exponents, self.value_exponents)

    def select(self, q, page_table, lengths, count: int, first: int = 1, last: int = 1):
        """The ``count`` pages of every sequence and key head that the queries can score highest with by their bounds (the sum over
        the head's queries), the ``first`` and ``last`` ones always among them; ascending, -1 behind them."""
        if self.bounds is None:
            raise RuntimeError("select: the cache keeps no bounds")
        return ops.select_pages(q, self.bounds, page_table, lengths, self.page_size, count, first, last)
