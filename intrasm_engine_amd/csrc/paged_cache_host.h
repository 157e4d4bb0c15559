// What the entry points of the paged cache share on the host.
#pragma once
#include "paged_cache_device.cuh"

namespace iex {

inline int log2_of(int power) {
  int shift = 0;
  while (1 << shift < power) ++shift;
  return shift;
}

// The cache's own arguments.  `written`: keys and values are needed (a selection reads the bounds only).
inline int check_paged_cache(const iex_paged_cache* c, const char* what, bool written) {
  IEX_REQUIRE(c, IEX_ERR_BAD_ARGUMENT, "%s: null pointer argument", what);
  IEX_REQUIRE(c->dtype == IEX_F16 || c->dtype == IEX_BF16, IEX_ERR_UNSUPPORTED, "%s: fp16 or bf16", what);
  IEX_REQUIRE(c->head_dim == 64 || c->head_dim == 128 || c->head_dim == 256, IEX_ERR_UNSUPPORTED, "%s: heads of 64, 128 or 256 (head_dim=%d)", what, c->head_dim);
  IEX_REQUIRE(c->page_size >= 16 && c->page_size <= 256 && (c->page_size & (c->page_size - 1)) == 0, IEX_ERR_UNSUPPORTED,
              "%s: pages of 16, 32, 64, 128 or 256 tokens (page_size=%d)", what, c->page_size);
  IEX_REQUIRE(c->pages >= 0 && c->kv_heads >= 0 && c->seqs >= 0 && c->table_width >= 0, IEX_ERR_BAD_ARGUMENT, "%s: negative dimension", what);
  IEX_REQUIRE((long long)c->table_width * c->page_size < (1ll << 30), IEX_ERR_TOO_LARGE, "%s: up to 2^30 tokens in a sequence's table (%d pages of %d)", what,
              c->table_width, c->page_size);
  IEX_REQUIRE(c->kv_heads <= 4096, IEX_ERR_TOO_LARGE, "%s: up to 4096 key heads", what);
  if (c->seqs == 0 || c->kv_heads == 0) return 0;
  IEX_REQUIRE(c->lengths && (c->table || c->table_width == 0), IEX_ERR_BAD_ARGUMENT, "%s: null pointer argument", what);
  if (c->pages == 0) return 0;
  if (!written) return 0;
  IEX_REQUIRE(c->keys && c->values && (!c->eight_bits || (c->key_exponents && c->value_exponents)), IEX_ERR_BAD_ARGUMENT, "%s: null pointer argument", what);
  const long long row = (long long)c->kv_heads * c->page_size * c->head_dim, chunk = c->eight_bits ? 16 : 8;
  IEX_REQUIRE(aligned(c->keys, 16) && aligned(c->values, 16) && c->key_page_stride % chunk == 0 && c->value_page_stride % chunk == 0 &&
                  (!c->eight_bits || (aligned(c->key_exponents, 16) && aligned(c->value_exponents, 16))) && aligned(c->bounds, 16),
              IEX_ERR_UNSUPPORTED, "%s: the cache's pages must be 16-byte aligned", what);
  IEX_REQUIRE(c->pages == 1 || (c->key_page_stride >= row && c->value_page_stride >= row), IEX_ERR_BAD_ARGUMENT, "%s: pages overlap", what);
  return 0;
}

// Rows of whole aligned 16-byte chunks.
inline bool rows_of_chunks(const void* x, const long long* strides) { return aligned(x, 16) && strides[2] == 1 && strides[0] % 8 == 0 && strides[1] % 8 == 0; }

inline PagedParams paged_params(const iex_paged_cache& c) {
  return PagedParams{c.pages, log2_of(c.page_size), c.kv_heads, c.seqs, c.table_width, c.key_page_stride, c.value_page_stride, c.table_stride,
                     c.keys, c.values, c.key_exponents, c.value_exponents, c.table, c.lengths};
}

}  // namespace iex
