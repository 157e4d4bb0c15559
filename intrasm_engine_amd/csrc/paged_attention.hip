// Host side of attention over a paged cache (paged_attention_device.cuh).
#include "paged_attention_host.h"

namespace iex {
namespace {

template <bool BF16, int D, bool E8, int WAVES>
struct Launch {
  static int run(const PagedAttentionParams& p, const Split& s, hipStream_t stream) {
    if (int rc = launch_attention<BF16, D, E8, WAVES, false>(p, s, stream)) return rc;
    if (s.fixed == 1) return 0;
    note_kernel("paged_join_kernel<%s, %d>", BF16 ? "bf16" : "f16", D);
    hipLaunchKernelGGL((paged_join_kernel<BF16, D, E8>), dim3((unsigned)p.cache.seqs, (unsigned)p.heads), dim3(256), 0, stream, p);
    return check_hip(hipGetLastError(), "paged attention join launch");
  }
};

}  // namespace
}  // namespace iex

extern "C" size_t iex_paged_attention_workspace_bytes(const iex_paged_cache* cache, int heads, int count) {
  using namespace iex;
  if (check_paged_cache(cache, "paged_attention", false) || check_heads(cache, heads, "paged_attention") || heads == 0 || cache->seqs == 0 || count < 0 ||
      (long long)count * cache->page_size >= kMostListed)
    return 0;
  const Split s = split_of(*cache, heads, count);
  if (s.fixed == 1) return 0;
  return partial_floats(*cache, s) * 4 + (size_t)s.workgroups * s.pitch * 8;
}

extern "C" int iex_paged_attention(const iex_paged_cache* cache, int heads, const void* q, const long long* q_strides, float scale, const int* listed, int count,
                                   void* out, const long long* out_strides, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace iex;
  trail_reset();
  if (int rc = check_paged_cache(cache, "paged_attention", true)) return rc;
  if (int rc = check_heads(cache, heads, "paged_attention")) return rc;
  IEX_REQUIRE(count >= 0 && (!listed || count > 0), IEX_ERR_BAD_ARGUMENT, "paged_attention: a list of pages must have entries");
  IEX_REQUIRE(listed || count == 0, IEX_ERR_BAD_ARGUMENT, "paged_attention: null pointer argument");
  IEX_REQUIRE((long long)count * cache->page_size < kMostListed, IEX_ERR_TOO_LARGE, "paged_attention: up to 2^30 tokens in a list of pages");
  if (cache->seqs == 0 || heads == 0) return 0;
  if (int rc = check_attention(cache, heads, q, q_strides, scale, out, out_strides, "paged_attention")) return rc;
  const Split s = split_of(*cache, heads, count);
  if (int rc = check_split(cache, heads, count, s, "paged_attention")) return rc;
  const size_t need = iex_paged_attention_workspace_bytes(cache, heads, count);
  IEX_REQUIRE(need == 0 || (workspace && aligned(workspace, 256) && workspace_bytes >= need), IEX_ERR_BAD_ARGUMENT,
              "paged_attention: needs a 256-byte aligned workspace of %zu bytes", need);
  const PagedAttentionParams p = attention_params(*cache, heads, q, q_strides, scale, listed, count, out, out_strides, workspace, s);
  return launch_form<Launch>(*cache, p, s, static_cast<hipStream_t>(stream));
}
