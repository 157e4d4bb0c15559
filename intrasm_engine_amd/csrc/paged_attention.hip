// Host side of attention over a paged cache (paged_attention_device.cuh).
#include "paged_attention_device.cuh"
#include "paged_cache_host.h"

namespace iex {
namespace {

// Workgroups that a launch aims at: what fills the chip's 256 CUs several times over, so that parts of unequal length even out.
constexpr int kPagedWorkgroups = 2048;

struct Split {
  long long slots, items, blocks;   // parts beyond one per sequence and block of heads, workgroups per block of heads, such blocks
  int pitch;
};
Split split_of(const iex_paged_cache& c, int heads, int count) {
  const int group = heads / c.kv_heads;
  Split s;
  s.blocks = (long long)c.kv_heads * ceil_div(group, 16);
  s.pitch = group < 16 ? group : 16;
  const long long wanted = kPagedWorkgroups / s.blocks;
  s.slots = paged_slots(wanted < 1 ? 1 : wanted, c.seqs, (long long)(count ? count : c.table_width) * c.page_size, kPagedLeast);
  s.items = c.seqs + s.slots;
  return s;
}
// (per part: rows x head_dim sums, then rows pairs)
size_t partial_floats(const iex_paged_cache& c, const Split& s) { return (size_t)s.items * s.blocks * s.pitch * c.head_dim; }

template <bool BF16, int D, bool E8>
int launch(const PagedAttentionParams& p, const Split& s, hipStream_t stream) {
  const int lds = kPagedWaves * s.pitch * (D + 2) * 4;
  auto kern = paged_attention_kernel<BF16, D, E8>;
  if (lds > 64 * 1024) {
    static thread_local bool raised = false;   // per instantiation
    if (!raised) {
      if (int rc = check_hip(hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, kPagedWaves * 16 * (D + 2) * 4),
                             "hipFuncSetAttribute(LDS size)"))
        return rc;
      raised = true;
    }
  }
  note_kernel("paged_attention_kernel<%s, %d, %s>", BF16 ? "bf16" : "f16", D, E8 ? "e4m3" : "16");
  hipLaunchKernelGGL(kern, dim3((unsigned)s.items, (unsigned)s.blocks), dim3(kPagedWaves * kWave), lds, stream, p);
  if (int rc = check_hip(hipGetLastError(), "paged attention launch")) return rc;
  if (s.slots == 0) return 0;
  note_kernel("paged_join_kernel<%s, %d>", BF16 ? "bf16" : "f16", D);
  hipLaunchKernelGGL((paged_join_kernel<BF16, D>), dim3((unsigned)p.cache.seqs, (unsigned)p.heads), dim3(256), 0, stream, p, (int)s.items);
  return check_hip(hipGetLastError(), "paged attention join launch");
}

template <bool BF16>
int launch_type(const PagedAttentionParams& p, const Split& s, int head_dim, bool e8, hipStream_t stream) {
  if (head_dim == 64) return e8 ? launch<BF16, 64, true>(p, s, stream) : launch<BF16, 64, false>(p, s, stream);
  if (head_dim == 128) return e8 ? launch<BF16, 128, true>(p, s, stream) : launch<BF16, 128, false>(p, s, stream);
  return e8 ? launch<BF16, 256, true>(p, s, stream) : launch<BF16, 256, false>(p, s, stream);
}

int check_heads(const iex_paged_cache* c, int heads, const char* what) {
  IEX_REQUIRE(heads >= 0, IEX_ERR_BAD_ARGUMENT, "%s: negative dimension", what);
  IEX_REQUIRE(c->kv_heads == 0 ? heads == 0 : heads % c->kv_heads == 0, IEX_ERR_BAD_ARGUMENT, "%s: query heads must be a multiple of key heads (%d, %d)", what, heads,
              c->kv_heads);
  return 0;
}

}  // namespace
}  // namespace iex

extern "C" size_t iex_paged_attention_workspace_bytes(const iex_paged_cache* cache, int heads, int count) {
  using namespace iex;
  if (check_paged_cache(cache, "paged_attention", false) || check_heads(cache, heads, "paged_attention") || heads == 0 || cache->seqs == 0 || count < 0) return 0;
  const Split s = split_of(*cache, heads, count);
  if (s.slots == 0) return 0;
  return partial_floats(*cache, s) * 4 + (size_t)s.items * s.blocks * s.pitch * 8;
}

extern "C" int iex_paged_attention(const iex_paged_cache* cache, int heads, const void* q, const long long* q_strides, float scale, const int* listed, int count,
                                   void* out, const long long* out_strides, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace iex;
  trail_reset();
  if (int rc = check_paged_cache(cache, "paged_attention", true)) return rc;
  if (int rc = check_heads(cache, heads, "paged_attention")) return rc;
  IEX_REQUIRE(count >= 0 && (!listed || count > 0), IEX_ERR_BAD_ARGUMENT, "paged_attention: a list of pages must have entries");
  IEX_REQUIRE(listed || count == 0, IEX_ERR_BAD_ARGUMENT, "paged_attention: null pointer argument");
  IEX_REQUIRE((long long)count * cache->page_size < (1ll << 30), IEX_ERR_TOO_LARGE, "paged_attention: up to 2^30 tokens in a list of pages");
  if (cache->seqs == 0 || heads == 0) return 0;
  IEX_REQUIRE(q && q_strides && out && out_strides, IEX_ERR_BAD_ARGUMENT, "paged_attention: null pointer argument");
  IEX_REQUIRE(aligned(q, 2) && aligned(out, 2), IEX_ERR_UNSUPPORTED, "paged_attention: operands must be aligned to their elements");
  IEX_REQUIRE(scale > 0.f && scale < 1e30f, IEX_ERR_UNSUPPORTED, "paged_attention: the scale must be positive and finite");
  const Split s = split_of(*cache, heads, count);
  const long long tiles = (long long)cache->seqs * paged_tiles((count ? count : cache->table_width) * cache->page_size);
  IEX_REQUIRE(tiles < (1ll << 31) && s.items < (1ll << 31) && s.blocks < 65536 && heads < 65536, IEX_ERR_TOO_LARGE, "paged_attention: too many sequences or heads");
  const size_t need = iex_paged_attention_workspace_bytes(cache, heads, count);
  IEX_REQUIRE(need == 0 || (workspace && aligned(workspace, 256) && workspace_bytes >= need), IEX_ERR_BAD_ARGUMENT,
              "paged_attention: needs a 256-byte aligned workspace of %zu bytes", need);
  PagedAttentionParams p{};
  p.cache = paged_params(*cache);
  p.heads = heads, p.group = heads / cache->kv_heads, p.group_tiles = ceil_div(p.group, 16), p.pitch = s.pitch;
  p.slots = (int)s.slots, p.count = count, p.listed = listed;
  p.q = static_cast<const unsigned short*>(q), p.out = static_cast<unsigned short*>(out);
  for (int i = 0; i < 3; ++i) p.q_strides[i] = q_strides[i], p.out_strides[i] = out_strides[i];
  p.scale_log2 = scale * 1.44269504088896340736f;
  p.partial = static_cast<float*>(workspace);
  p.stats = p.partial + (need ? partial_floats(*cache, s) : 0);
  hipStream_t st = static_cast<hipStream_t>(stream);
  return cache->dtype == IEX_BF16 ? launch_type<true>(p, s, cache->head_dim, cache->eight_bits, st) : launch_type<false>(p, s, cache->head_dim, cache->eight_bits, st);
}
