"""A paged cache of keys and values for generation: tokens appended to it, single new tokens attending to it, pages selected, tokens
dropped that got least attention.

Operators under ``torch.ops.iex_ops`` (``csrc/host/paged_ops.h``), on the current stream, capturable, without a gradient but for
``rotate``'s of x (its table has none: a table that requires one is refused), none with forward mode (dual tensors are refused):

    kv_append_(k, v, keys, values, page_table, lengths, offsets=None, q=None, rotation=None, interleaved=False, bounds=None,
               key_exponents=None, value_exponents=None, positions=None, sections=None, in_turn=False) -> q, rotated (None without q)
    rotate(x, rotation, positions, sections=None, in_turn=False, interleaved=False, back=False) -> x, rotated (fp32, fp16, bf16)
    paged_attention(q, keys, values, page_table, lengths, scale=None, pages=None, key_exponents=None, value_exponents=None)
    paged_attention_accumulate_(q, keys, values, page_table, lengths, weights, scale=None, key_exponents=None, value_exponents=None)
    select_pages(q, bounds, page_table, lengths, page_size, count, first=1, last=1) -> (sequences, kv_heads, count) int32
    evict_tokens_(keys, values, page_table, lengths, weights, keep, recent, first=0, bounds=None, key_exponents=None,
                  value_exponents=None) -> (sequences, kv_heads, keep) int32

Tokens are (tokens, heads, head_dim) tensors of fp16 or bf16 with any strides; what comes back has the strides of ``q``, so the
(heads * head_dim, tokens) matrices that projections ``W @ X`` leave and take go in as ``x.view(heads, head_dim, tokens).permute(2, 0,
1)`` and come out the same way.  ``page_table``: (sequences, width) int32, the pages of every sequence in order; ``lengths``:
(sequences) int32, tokens of every sequence, the new ones of an append counted.  Both are read on the device when the kernels
run: a captured graph follows what they hold at each replay.  A length is cut to what the table holds; a page outside
the cache (-1, say) counts as given back: nothing is written to it, nothing of it is attended to, it is not selected.

``positions``: (tokens) or (axes, tokens) int32, on the device, where tokens are for their rotation: on up to four axes (time, height and width of
pictures and videos), ``sections`` saying how many of the rotation's planes go by each axis, one stretch behind the other or, ``in_turn``, dealt in turn as
long as an axis has planes left.  Without them a token's position is its place in its sequence, which it no longer is once tokens before it
have been dropped.  A position below 0 counts as 0; behind the rotation's rows the planes of its axis come out as NaN.

``weights``: (sequences, kv_heads, tokens of a table) float32, zeros at first, what every token got of attention so far: each pass adds the sum of the
softmax weights of a key head's queries.  They belong to the rows of ``page_table``, not to pages, so sequences may share pages; the weights of
tokens that are taken back (a shorter length) are the caller's to clear.

:class:`KVCache` holds a cache's tensors and calls them.
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

    def new_weights(self, page_table):
        """An account, empty, for :meth:`attend` and :meth:`evict_`: what the tokens of a table's sequences got of attention."""
        return torch.zeros(page_table.shape[0], self.kv_heads, page_table.shape[1] * self.page_size, dtype=torch.float32, device=self.keys.device)

    def fits(self, weights, page_table) -> bool:
        """Whether ``weights`` are an account for this table's sequences."""
        shape = (page_table.shape[0], self.kv_heads, page_table.shape[1] * self.page_size)
        return (tuple(weights.shape) == shape and weights.dtype == torch.float32 and weights.is_contiguous() and weights.device == self.keys.device
                and weights.data_ptr() % 16 == 0 and not (torch.is_grad_enabled() and weights.requires_grad))

    def append_(self, k, v, page_table, lengths, offsets=None, q=None, rotation=None, interleaved: bool = False, positions=None, sections=None, in_turn: bool = False):
        """Write the newest tokens' keys and values, (tokens, kv_heads, head_dim): token s is sequence s's, or ``offsets[s] ..
        offsets[s + 1]`` are (int32, from 0).  Keys and ``q`` are rotated by ``rotation`` (:func:`rotation_table`; a row for every
        position that the table can hold) at their positions, or at ``positions`` (a row for each of them).  Returns q so."""
        return ops.kv_append_(k, v, self.keys, self.values, page_table, lengths, offsets, q, rotation, interleaved, self.bounds, self.key_exponents,
                              self.value_exponents, positions, sections, in_turn)

    def attend(self, q, page_table, lengths, scale: float | None = None, pages=None, weights=None):
        """softmax(scale q k^T) v over each sequence's tokens, or those of its listed ``pages`` (:meth:`select`); q: (sequences, heads,
        head_dim), heads a multiple of ``kv_heads``; ``scale``: 1 / sqrt(head_dim).  ``weights`` (:meth:`new_weights`; every page is attended
        to then): what tokens get is added to them."""
        if weights is not None:
            if pages is not None:
                raise ValueError("attend: an account is kept over all pages, not over listed ones")
            return ops.paged_attention_accumulate_(q, self.keys, self.values, page_table, lengths, weights, scale, self.key_exponents, self.value_exponents)
        return ops.paged_attention(q, self.keys, self.values, page_table, lengths, scale, pages, self.key_exponents, self.value_exponents)

    def select(self, q, page_table, lengths, count: int, first: int = 1, last: int = 1):
        """The ``count`` pages of every sequence and key head that the queries can score highest with by their bounds (the sum over
        the head's queries), the ``first`` and ``last`` ones always among them; ascending, -1 behind them."""
        if self.bounds is None:
            raise RuntimeError("select: the cache keeps no bounds")
        return ops.select_pages(q, self.bounds, page_table, lengths, self.page_size, count, first, last)

    def evict_(self, page_table, lengths, weights, keep: int, recent: int, first: int = 0):
        """Sequences of more than ``keep`` tokens lose those that got least: of every key head's the ``first``, the ``recent`` and the ones with the
        largest ``weights`` stay (of two that are equal the earlier) and move up, in order, within the sequence's own pages, which it must share
        with nobody; ``lengths``, ``weights`` and bounds follow.  ``lengths`` are cut in place: the caches of several layers, which go by one ``lengths``, are
        cut by a copy each (``lengths.clone()``) but the last, else the first leaves nothing to do to the others.  Returns where they were, (sequences, kv_heads, keep), -1 behind shorter sequences.  New
        tokens then need ``positions`` of their own.  A sequence with pages given back is passed over (all -1).  Pages that no sequence needs any
        more are the caller's to give to others.  (-2, and NaN in the cache: rows whose move was given up, as graphs that share memory can make it if they
        are replayed at the same time.)"""
        return ops.evict_tokens_(self.keys, self.values, page_table, lengths, weights, keep, recent, first, self.bounds, self.key_exponents, self.value_exponents)
