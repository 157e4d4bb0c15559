// Host side of attention over a paged cache that keeps account: what every token got of the queries' attention is added up (paged_attention_device.cuh).
#include "paged_attention_host.h"

namespace iex {
namespace {

constexpr int kMostGroup = 4096;   // query heads of a key head: their shares are in LDS

// Whole rows whose queries are together add their weights where they are, in the launch that has them.
bool at_once(const Split& s, int group) { return s.fixed == 1 && group <= 16; }

// Workgroups that take turns at the tokens of a sequence and key head: as many as the table can have work for, and no more than the chip has room
// for (eight of 256 threads on each CU).
int account_side(const iex_paged_cache& c) {
  const long long rows = (long long)c.seqs * c.kv_heads, most = ceil_div((long long)c.table_width * c.page_size, kAccountTokens), room = 2048 / rows;
  const long long side = most < room ? most : room;
  return side < 1 ? 1 : (int)side;
}

template <bool BF16, int D, bool E8, int WAVES>
struct Launch {
  static int run(const PagedAttentionParams& p, const Split& s, int side, hipStream_t stream) {
    if (int rc = launch_attention<BF16, D, E8, WAVES, true>(p, s, stream)) return rc;
    if (p.at_once) return 0;
    const int joins = s.fixed == 1 ? 0 : p.cache.seqs * p.heads;
    note_kernel("paged_account_kernel<%s, %d>", BF16 ? "bf16" : "f16", D);
    hipLaunchKernelGGL((paged_account_kernel<BF16, D, E8>), dim3((unsigned)joins + (unsigned)p.cache.seqs * p.cache.kv_heads * side), dim3(256), p.group * 8, stream, p, joins,
                       side);
    return check_hip(hipGetLastError(), "paged attention account launch");
  }
};

// The workspace: parts' sums and statistics (rows that are cut), rows' statistics, scores.
size_t parts_bytes(const iex_paged_cache& c, const Split& s) { return s.fixed == 1 ? 0 : (partial_floats(c, s) * 4 + (size_t)s.workgroups * s.pitch * 8 + 255) / 256 * 256; }
size_t rows_bytes(const iex_paged_cache& c, int heads) { return ((size_t)c.seqs * heads * 8 + 255) / 256 * 256; }
size_t scores_bytes(const iex_paged_cache& c, int heads) { return (size_t)c.seqs * heads * c.table_width * c.page_size * 4; }

}  // namespace
}  // namespace iex

extern "C" size_t iex_paged_attention_accumulate_workspace_bytes(const iex_paged_cache* cache, int heads) {
  using namespace iex;
  if (check_paged_cache(cache, "paged_attention_accumulate", false) || check_heads(cache, heads, "paged_attention_accumulate") || heads == 0 || cache->seqs == 0) return 0;
  return parts_bytes(*cache, split_of(*cache, heads, 0)) + rows_bytes(*cache, heads) + scores_bytes(*cache, heads);
}

extern "C" int iex_paged_attention_accumulate(const iex_paged_cache* cache, int heads, const void* q, const long long* q_strides, float scale, float* weights, void* out,
                                              const long long* out_strides, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace iex;
  constexpr const char* what = "paged_attention_accumulate";
  trail_reset();
  if (int rc = check_paged_cache(cache, what, true)) return rc;
  if (int rc = check_heads(cache, heads, what)) return rc;
  if (cache->seqs == 0 || heads == 0) return 0;
  if (int rc = check_attention(cache, heads, q, q_strides, scale, out, out_strides, what)) return rc;
  IEX_REQUIRE(weights || cache->table_width == 0, IEX_ERR_BAD_ARGUMENT, "%s: null pointer argument", what);
  IEX_REQUIRE(aligned(weights, 16), IEX_ERR_UNSUPPORTED, "%s: the weights must be 16-byte aligned", what);
  IEX_REQUIRE(heads / cache->kv_heads <= kMostGroup, IEX_ERR_TOO_LARGE, "%s: up to %d query heads of a key head", what, kMostGroup);
  const Split s = split_of(*cache, heads, 0);
  if (int rc = check_split(cache, heads, 0, s, what)) return rc;
  const int side = account_side(*cache);
  IEX_REQUIRE((long long)cache->seqs * heads + (long long)cache->seqs * cache->kv_heads * side < (1ll << 24), IEX_ERR_TOO_LARGE, "%s: too many sequences or heads", what);
  const size_t need = iex_paged_attention_accumulate_workspace_bytes(cache, heads);
  IEX_REQUIRE(workspace && aligned(workspace, 256) && workspace_bytes >= need, IEX_ERR_BAD_ARGUMENT, "%s: needs a 256-byte aligned workspace of %zu bytes", what, need);
  PagedAttentionParams p = attention_params(*cache, heads, q, q_strides, scale, nullptr, 0, out, out_strides, workspace, s);
  char* const after = static_cast<char*>(workspace) + parts_bytes(*cache, s);
  p.weights = weights;
  p.row_stats = reinterpret_cast<float*>(after);
  p.scores = reinterpret_cast<float*>(after + rows_bytes(*cache, heads));
  p.at_once = at_once(s, p.group);
  return launch_form<Launch>(*cache, p, s, side, static_cast<hipStream_t>(stream));
}
