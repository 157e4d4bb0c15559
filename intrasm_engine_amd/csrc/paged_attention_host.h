// What the two attentions over a paged cache share on the host: how rows are cut, and the launch of their kernel.
#pragma once
#include "paged_attention_device.cuh"
#include "paged_cache_host.h"

#include <climits>

namespace iex {
namespace {

// Workgroups of four wavefronts that are resident at once: by their registers two to four on each of the 256 CUs.
int resident(int head_dim) { return 256 * paged_simd_waves(head_dim); }

// Rows of up to this many tiles stay whole, and there is no second launch: 128 rows of 700 tokens of 128 12.0 us, cut 17.0; 512 of 600 .. 1023
// 37.4 and 43; 32 of 2000, the other side, 13.2 cut and 22.8 whole.  (Where all tiles of shorter rows could have a workgroup each, cutting would be
// the faster, which the rule leaves: 32 of 700 11.1 whole and 10.0 cut.)
constexpr int kWholeTiles = 8;
// Whole rows go to eight wavefronts each where four would leave CUs without work: 128 rows of 700 12.0 us by eight, 16.0 by four; 512 of
// 500 28.1 and 23.7.
constexpr int kWideRows = 512;
// Rows of up to this many tokens have a wavefront each: 4096 rows of 12 tokens in tables of 64 28.6 us by four, 14.3 by one; of 64 33.3 and
// 24.9; of 128, the other side, 47.5 and 51.5.
constexpr int kNarrow = 64;
// Parts: one round of resident workgroups where rows are few (131071 tokens, 8 rows: 92.5 us, two rounds 101.6), two where rows of unequal
// lengths come anyway (512 rows of 4000 .. 16384, e4m3: 236 one, 206.5 two; 2048 of 1 .. 4096, heads of 64: 65.5 and 61.9; three and four rounds
// as two).
constexpr int kTwoRounds = 256;
// Tiles have a workgroup each, if that makes at most this many, one on each CU: a sequence of 4000 tokens, 8 key heads of 64 (256 workgroups)
// 12.0 us, by two tiles 13.6; 64 listed pages of 64 (256) 10.3 and 11.9; 8192 tokens (512), the other side, 16.4 and 14.8.
constexpr int kFew = 256;
constexpr long long kMostListed = 1ll << 30;   // tokens of a list of pages

struct Split {
  long long blocks, slots, workgroups;   // blocks of up to 16 heads of a key head; parts beyond one per sequence; workgroups of the launch
  int few, fixed, pitch;                 // (PagedAttentionParams); parts of every row (0: by the lengths)
  bool wide, narrow;
};
Split split_of(const iex_paged_cache& c, int heads, int count) {
  const int group = heads / c.kv_heads, most = paged_tiles((count ? count : c.table_width) * c.page_size);
  Split s;
  s.blocks = (long long)c.kv_heads * ceil_div(group, 16);
  s.pitch = group < 16 ? group : 16;
  const long long rows = s.blocks * c.seqs;
  const bool whole = most <= kWholeTiles;
  s.narrow = (count ? count : c.table_width) * c.page_size <= kNarrow;
  s.wide = whole && rows < kWideRows;
  const int round = resident(c.head_dim), wanted = rows < kTwoRounds ? round : 2 * round;
  s.slots = whole ? 0 : paged_slots(wanted / s.blocks, c.seqs, most);
  s.few = (int)(kFew / s.blocks);
  s.fixed = whole ? 1 : 0;
  if (count && !whole) {   // (every row is as long)
    const long long all = (long long)c.seqs * most;
    const int total = all < INT_MAX ? (int)all : INT_MAX;
    s.fixed = paged_parts(most, paged_part_most(total - c.seqs, (int)s.slots, paged_least(total, s.few)));
  }
  s.workgroups = s.blocks * (s.fixed ? (long long)c.seqs * s.fixed : c.seqs + s.slots);
  return s;
}
// (per part: rows x head_dim sums, then rows pairs)
size_t partial_floats(const iex_paged_cache& c, const Split& s) { return (size_t)s.workgroups * s.pitch * c.head_dim; }

// LDS: the wavefronts' sums, maxima and sums of weights; the shares of the queries.
inline int attention_lds(int pitch, int head_dim, int waves, bool weigh) {
  return waves * pitch * (paged_sum_pitch(head_dim) + 2) * 4 + (weigh ? (2 * pitch + 1) * 4 : 0);
}
template <bool BF16, int D, bool E8, int WAVES, bool WEIGH>
int launch_attention(const PagedAttentionParams& p, const Split& s, hipStream_t stream) {
  const int lds = attention_lds(s.pitch, D, WAVES, WEIGH);
  auto kern = paged_attention_kernel<BF16, D, E8, WAVES, WEIGH>;
  if (lds > 64 * 1024) {
    static thread_local unsigned long long raised = 0;   // per instantiation: on which devices
    int device = 0;
    if (int rc = check_hip(hipGetDevice(&device), "hipGetDevice")) return rc;
    if (!(raised >> (device & 63) & 1)) {
      if (int rc = check_hip(hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, attention_lds(16, D, WAVES, WEIGH)),
                             "hipFuncSetAttribute(LDS size)"))
        return rc;
      raised |= 1ull << (device & 63);
    }
  }
  note_kernel("paged_attention_kernel<%s, %d, %s, %d>%s", BF16 ? "bf16" : "f16", D, E8 ? "e4m3" : "16", WAVES, WEIGH ? " (scores kept)" : "");
  hipLaunchKernelGGL(kern, dim3((unsigned)s.workgroups), dim3(WAVES * kWave), lds, stream, p);
  return check_hip(hipGetLastError(), "paged attention launch");
}

int check_heads(const iex_paged_cache* c, int heads, const char* what) {
  IEX_REQUIRE(heads >= 0, IEX_ERR_BAD_ARGUMENT, "%s: negative dimension", what);
  IEX_REQUIRE(c->kv_heads == 0 ? heads == 0 : heads % c->kv_heads == 0, IEX_ERR_BAD_ARGUMENT, "%s: query heads must be a multiple of key heads (%d, %d)", what, heads,
              c->kv_heads);
  return 0;
}


// The arguments that both have, beyond the cache's.
int check_attention(const iex_paged_cache* cache, int heads, const void* q, const long long* q_strides, float scale, const void* out, const long long* out_strides,
                    const char* what) {
  IEX_REQUIRE(cache->pages > 0, IEX_ERR_BAD_ARGUMENT, "%s: a cache without pages", what);
  IEX_REQUIRE(q && q_strides && out && out_strides, IEX_ERR_BAD_ARGUMENT, "%s: null pointer argument", what);
  IEX_REQUIRE(aligned(q, 2) && aligned(out, 2), IEX_ERR_UNSUPPORTED, "%s: operands must be aligned to their elements", what);
  IEX_REQUIRE(scale > 0.f && scale < 1e30f, IEX_ERR_UNSUPPORTED, "%s: the scale must be positive and finite", what);
  return 0;
}
int check_split(const iex_paged_cache* cache, int heads, int count, const Split& s, const char* what) {
  const long long tiles = (long long)cache->seqs * paged_tiles((count ? count : cache->table_width) * cache->page_size);
  IEX_REQUIRE(tiles < (1ll << 31) && s.workgroups < (1ll << 30) && heads < 65536, IEX_ERR_TOO_LARGE, "%s: too many sequences or heads", what);
  return 0;
}

// `workspace`: the parts' sums, then their statistics.
inline PagedAttentionParams attention_params(const iex_paged_cache& cache, int heads, const void* q, const long long* q_strides, float scale, const int* listed, int count,
                                             void* out, const long long* out_strides, void* workspace, const Split& s) {
  PagedAttentionParams p{};
  p.cache = paged_params(cache);
  p.heads = heads, p.group = heads / cache.kv_heads, p.group_tiles = ceil_div(p.group, 16), p.pitch = s.pitch;
  p.count = count, p.listed = listed, p.blocks = (int)s.blocks, p.slots = (int)s.slots, p.few = s.few, p.fixed = s.fixed;
  p.q = static_cast<const unsigned short*>(q), p.out = static_cast<unsigned short*>(out);
  for (int i = 0; i < 3; ++i) p.q_strides[i] = q_strides[i], p.out_strides[i] = out_strides[i];
  p.q_rows = rows_of_chunks(q, q_strides);
  p.scale_log2 = scale * 1.44269504088896340736f;
  p.partial = static_cast<float*>(workspace);
  p.stats = s.fixed == 1 ? p.partial : p.partial + partial_floats(cache, s);
  return p;
}

// LAUNCH<bf16, head_dim, e4m3, wavefronts> by the cache's types and the split.
template <template <bool, int, bool, int> class LAUNCH, bool BF16, int D, bool E8, typename... MORE>
int launch_waves(const PagedAttentionParams& p, const Split& s, MORE... more) {
  if (s.narrow) return LAUNCH<BF16, D, E8, 1>::run(p, s, more...);
  return s.wide ? LAUNCH<BF16, D, E8, 8>::run(p, s, more...) : LAUNCH<BF16, D, E8, 4>::run(p, s, more...);
}
template <template <bool, int, bool, int> class LAUNCH, bool BF16, typename... MORE>
int launch_dim(const iex_paged_cache& c, const PagedAttentionParams& p, const Split& s, MORE... more) {
  if (c.head_dim == 64) return c.eight_bits ? launch_waves<LAUNCH, BF16, 64, true>(p, s, more...) : launch_waves<LAUNCH, BF16, 64, false>(p, s, more...);
  if (c.head_dim == 128) return c.eight_bits ? launch_waves<LAUNCH, BF16, 128, true>(p, s, more...) : launch_waves<LAUNCH, BF16, 128, false>(p, s, more...);
  return c.eight_bits ? launch_waves<LAUNCH, BF16, 256, true>(p, s, more...) : launch_waves<LAUNCH, BF16, 256, false>(p, s, more...);
}
template <template <bool, int, bool, int> class LAUNCH, typename... MORE>
int launch_form(const iex_paged_cache& c, const PagedAttentionParams& p, const Split& s, MORE... more) {
  return c.dtype == IEX_BF16 ? launch_dim<LAUNCH, true>(c, p, s, more...) : launch_dim<LAUNCH, false>(c, p, s, more...);
}

}  // namespace
}  // namespace iex
