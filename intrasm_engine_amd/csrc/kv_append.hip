// Host side of appending to a paged cache (kv_append_device.cuh).
#include "kv_append_host.h"
#include "rotation_host.h"

namespace iex {
namespace {

// Features whose tokens are whole aligned 16-byte chunks (up to the last ones).  (At other alignments 16 bytes a lane cost more than two:
// 5 x 1001 tokens of 32 + 2 x 8 heads 67 us against 43.)
bool columns_of_chunks(const void* x, const long long* strides) { return aligned(x, 16) && strides[0] == 1 && strides[1] % 8 == 0 && strides[2] % 8 == 0; }

}  // namespace

int launch_kv_append(const iex_paged_cache& c, const AppendParams& p, bool rows, bool interleaved, hipStream_t s) { return launch_append<false>(c, p, rows, interleaved, s); }

}  // namespace iex

extern "C" int iex_kv_append_at(const iex_paged_cache* cache, int tokens, const int* offsets, int heads, const void* k, const long long* k_strides, const void* v,
                                const long long* v_strides, const void* q, const long long* q_strides, void* q_out, const long long* q_out_strides,
                                const iex_rotation* rotation, void* stream) {
  using namespace iex;
  trail_reset();
  if (int rc = check_paged_cache(cache, "kv_append", true)) return rc;
  IEX_REQUIRE(tokens >= 0 && heads >= 0, IEX_ERR_BAD_ARGUMENT, "kv_append: negative dimension");
  IEX_REQUIRE(offsets || tokens == cache->seqs, IEX_ERR_BAD_ARGUMENT, "kv_append: one token per sequence without offsets (%d tokens, %d sequences)", tokens, cache->seqs);
  if (tokens == 0) return 0;
  IEX_REQUIRE(k && v && k_strides && v_strides, IEX_ERR_BAD_ARGUMENT, "kv_append: null pointer argument");
  IEX_REQUIRE(heads == 0 || (q && q_out && q_strides && q_out_strides), IEX_ERR_BAD_ARGUMENT, "kv_append: null pointer argument");
  IEX_REQUIRE(cache->seqs == 0 || cache->lengths, IEX_ERR_BAD_ARGUMENT, "kv_append: null pointer argument");   // (without key heads too: queries turn by them)
  AppendParams p{};
  if (int rc = check_rotation(rotation, "kv_append", p.rotation)) return rc;
  const int rotary = p.rotation.features;
  IEX_REQUIRE(rotary % 16 == 0 && rotary <= cache->head_dim, IEX_ERR_UNSUPPORTED,
              "kv_append: rotated features must be a multiple of 16 of the head's (%d of %d)", rotary, cache->head_dim);
  IEX_REQUIRE(rotary == 0 || p.rotation.positions || (long long)p.rotation.rows >= (long long)cache->table_width * cache->page_size, IEX_ERR_BAD_ARGUMENT,
              "kv_append: the rotation must have a row for every position of the table (%d of %lld)", p.rotation.rows, (long long)cache->table_width * cache->page_size);
  IEX_REQUIRE(aligned(k, 2) && aligned(v, 2) && (heads == 0 || (aligned(q, 2) && aligned(q_out, 2))), IEX_ERR_UNSUPPORTED, "kv_append: operands must be aligned to their elements");
  p.cache = paged_params(*cache);
  p.tokens = tokens, p.heads = heads, p.offsets = offsets;
  auto operand = [](const void* x, const long long* strides) { return AppendOperand{static_cast<const unsigned short*>(x), strides[0], strides[1], strides[2]}; };
  p.k = operand(k, k_strides), p.v = operand(v, v_strides);
  if (heads) {
    p.q = operand(q, q_strides), p.q_out = static_cast<unsigned short*>(q_out);
    p.out_token = q_out_strides[0], p.out_head = q_out_strides[1], p.out_feature = q_out_strides[2];
  }
  p.bounds = static_cast<unsigned short*>(cache->bounds);
  const bool rows = rows_of_chunks(k, k_strides) && rows_of_chunks(v, v_strides) && (heads == 0 || (rows_of_chunks(q, q_strides) && rows_of_chunks(q_out, q_out_strides)));
  p.columns = columns_of_chunks(k, k_strides) && columns_of_chunks(v, v_strides) &&
              (heads == 0 || (columns_of_chunks(q, q_strides) && columns_of_chunks(q_out, q_out_strides)));
  const long long spans = offsets ? append_most_spans(tokens, cache->seqs, append_span(cache->page_size)) : tokens;
  // one head to a workgroup until there are workgroups enough, then four: they share what they read of the rotation (16 x 512 tokens of
  // 32 + 2 x 8 heads 44.3 us by one, 40.3 by four, 45.9 by eight; 64 x 2000 691, 676, 746; 4 x 512 tokens, the other side, 17.4, 18.2, 18.3)
  const long long all = spans * (2ll * cache->kv_heads + heads);
  p.per_group = all >= 4096 ? 4 : 1;
  IEX_REQUIRE(spans < (1ll << 31) && 2ll * cache->kv_heads + heads < 65536, IEX_ERR_TOO_LARGE, "kv_append: too many tokens or heads");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool interleaved = rotation && rotation->interleaved;
  return p.rotation.positions ? launch_kv_append_at(*cache, p, rows, interleaved, s) : launch_kv_append(*cache, p, rows, interleaved, s);
}

extern "C" int iex_kv_append(const iex_paged_cache* cache, int tokens, const int* offsets, int heads, const void* k, const long long* k_strides, const void* v,
                             const long long* v_strides, const void* q, const long long* q_strides, void* q_out, const long long* q_out_strides,
                             const float* rotation, int positions, int rotary, int interleaved, void* stream) {
  const iex_rotation by_place{rotation, positions, rotary, nullptr, 0, 1, nullptr, 0, interleaved};
  return iex_kv_append_at(cache, tokens, offsets, heads, k, k_strides, v, v_strides, q, q_strides, q_out, q_out_strides, &by_place, stream);
}
