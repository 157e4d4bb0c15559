// Host side of appending to a paged cache (kv_append_device.cuh).
#include "kv_append_device.cuh"
#include "paged_cache_host.h"

namespace iex {
namespace {

template <bool BF16, int D, bool E8, bool STAGED>
int launch(const AppendParams& p, bool interleaved, dim3 grid, hipStream_t stream) {
  note_kernel("kv_append_kernel<%s, %d, %s, %s, %s>", BF16 ? "bf16" : "f16", D, E8 ? "e4m3" : "16", STAGED ? "staged" : "rows", interleaved ? "interleaved" : "halves");
  if (interleaved) hipLaunchKernelGGL((kv_append_kernel<BF16, D, E8, STAGED, true>), grid, dim3(256), 0, stream, p);
  else hipLaunchKernelGGL((kv_append_kernel<BF16, D, E8, STAGED, false>), grid, dim3(256), 0, stream, p);
  return check_hip(hipGetLastError(), "kv_append launch");
}

template <bool BF16, int D>
int launch_forms(const AppendParams& p, bool e8, bool staged, bool interleaved, dim3 grid, hipStream_t s) {
  if (e8) return staged ? launch<BF16, D, true, true>(p, interleaved, grid, s) : launch<BF16, D, true, false>(p, interleaved, grid, s);
  return staged ? launch<BF16, D, false, true>(p, interleaved, grid, s) : launch<BF16, D, false, false>(p, interleaved, grid, s);
}

}  // namespace
}  // namespace iex

extern "C" int iex_kv_append(const iex_paged_cache* cache, int tokens, const int* offsets, int heads, const void* k, const long long* k_strides, const void* v,
                             const long long* v_strides, const void* q, const long long* q_strides, void* q_out, const long long* q_out_strides,
                             const float* rotation, int positions, int rotary, int interleaved, void* stream) {
  using namespace iex;
  trail_reset();
  if (int rc = check_paged_cache(cache, "kv_append", true)) return rc;
  IEX_REQUIRE(tokens >= 0 && heads >= 0, IEX_ERR_BAD_ARGUMENT, "kv_append: negative dimension");
  IEX_REQUIRE(offsets || tokens == cache->seqs, IEX_ERR_BAD_ARGUMENT, "kv_append: one token per sequence without offsets (%d tokens, %d sequences)", tokens, cache->seqs);
  if (tokens == 0) return 0;
  IEX_REQUIRE(k && v && k_strides && v_strides, IEX_ERR_BAD_ARGUMENT, "kv_append: null pointer argument");
  IEX_REQUIRE(heads == 0 || (q && q_out && q_strides && q_out_strides), IEX_ERR_BAD_ARGUMENT, "kv_append: null pointer argument");
  IEX_REQUIRE(rotary == 0 || (rotation && aligned(rotation, 16)), IEX_ERR_BAD_ARGUMENT, "kv_append: the rotation must be a 16-byte aligned array");
  IEX_REQUIRE(rotary >= 0 && rotary % 16 == 0 && rotary <= cache->head_dim, IEX_ERR_UNSUPPORTED,
              "kv_append: rotated features must be a multiple of 16 of the head's (%d of %d)", rotary, cache->head_dim);
  IEX_REQUIRE(rotary == 0 || (long long)positions >= (long long)cache->table_width * cache->page_size, IEX_ERR_BAD_ARGUMENT,
              "kv_append: the rotation must have a row for every position of the table (%d of %lld)", positions, (long long)cache->table_width * cache->page_size);
  IEX_REQUIRE(aligned(k, 2) && aligned(v, 2) && (heads == 0 || (aligned(q, 2) && aligned(q_out, 2))), IEX_ERR_UNSUPPORTED, "kv_append: operands must be aligned to their elements");
  AppendParams p{};
  p.cache = paged_params(*cache);
  p.tokens = tokens, p.heads = heads, p.rotary = rotary, p.offsets = offsets, p.rotation = rotation;
  p.k = static_cast<const unsigned short*>(k), p.v = static_cast<const unsigned short*>(v);
  p.q = static_cast<const unsigned short*>(q), p.q_out = static_cast<unsigned short*>(q_out);
  p.bounds = static_cast<unsigned short*>(cache->bounds);
  for (int i = 0; i < 3; ++i) {
    p.k_strides[i] = k_strides[i], p.v_strides[i] = v_strides[i];
    if (heads) p.q_strides[i] = q_strides[i], p.out_strides[i] = q_out_strides[i];
  }
  const bool staged = !(rows_of_chunks(k, k_strides) && rows_of_chunks(v, v_strides) && (heads == 0 || (rows_of_chunks(q, q_strides) && rows_of_chunks(q_out, q_out_strides))));
  const long long spans = offsets ? append_most_spans(tokens, cache->seqs, append_span(cache->page_size)) : tokens;
  // one head to a workgroup until there are workgroups enough; then as many as share what they read of the rotation
  const long long all = spans * (2ll * cache->kv_heads + heads);
  p.per_group = all > 8 * 2048 ? 8 : all > 2048 ? (int)(all / 2048) : 1;
  const int kv_groups = ceil_div(cache->kv_heads, p.per_group);
  const long long groups = (cache->bounds ? cache->kv_heads : kv_groups) + kv_groups + ceil_div(heads, p.per_group);
  IEX_REQUIRE(spans < (1ll << 31) && groups < 65536, IEX_ERR_TOO_LARGE, "kv_append: too many tokens or heads");
  const dim3 grid((unsigned)spans, (unsigned)groups);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool e8 = cache->eight_bits;
  if (cache->dtype == IEX_BF16) {
    if (cache->head_dim == 64) return launch_forms<true, 64>(p, e8, staged, interleaved, grid, s);
    if (cache->head_dim == 128) return launch_forms<true, 128>(p, e8, staged, interleaved, grid, s);
    return launch_forms<true, 256>(p, e8, staged, interleaved, grid, s);
  }
  if (cache->head_dim == 64) return launch_forms<false, 64>(p, e8, staged, interleaved, grid, s);
  if (cache->head_dim == 128) return launch_forms<false, 128>(p, e8, staged, interleaved, grid, s);
  return launch_forms<false, 256>(p, e8, staged, interleaved, grid, s);
}
