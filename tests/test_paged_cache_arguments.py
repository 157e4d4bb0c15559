"""Arguments of the paged cache's C entry points that are refused before anything is launched (no GPU: addresses that nothing stands behind)."""
import ctypes

import pytest

from intrasm_engine_amd import _lib

A = 4096
STRIDES = (ctypes.c_longlong * 3)(256, 128, 1)


def cache(**other):
    c = _lib.PagedCache(dtype=_lib.F16, eight_bits=0, pages=10, page_size=64, kv_heads=2, head_dim=128, key_page_stride=2 * 64 * 128, value_page_stride=2 * 64 * 128,
                        keys=A, values=A, table=A, seqs=3, table_width=4, table_stride=4, lengths=A)
    for name, value in other.items():
        setattr(c, name, value)
    return c


@pytest.mark.parametrize("offsets", [None, A])
def test_queries_alone_need_lengths(offsets):
    """A cache without key heads has no keys to place, but its queries are turned by their positions, which the lengths tell."""
    c = cache(kv_heads=0, lengths=None)
    rc = _lib.load().iex_kv_append(ctypes.byref(c), 3, offsets, 2, A, STRIDES, A, STRIDES, A, STRIDES, A, STRIDES, A, 256, 128, 0, None)
    assert rc == -1 and "null" in _lib.last_error()


@pytest.mark.parametrize("count,page_size", [((1 << 25) + (1 << 14), 256), (1 << 26, 16), ((1 << 30) + 4096, 64)])
def test_lists_that_are_refused_need_no_workspace(count, page_size):
    """2^30 tokens and more (sizes that pass 32 bits among them)."""
    lib, c = _lib.load(), cache(page_size=page_size, key_page_stride=2 * 256 * 128, value_page_stride=2 * 256 * 128)
    assert lib.iex_paged_attention_workspace_bytes(ctypes.byref(c), 4, count) == 0
    assert lib.iex_paged_attention(ctypes.byref(c), 4, A, STRIDES, 0.1, A, count, A, STRIDES, A, 1 << 40, None) == -3 and "2^30" in _lib.last_error()
