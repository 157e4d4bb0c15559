// Pages of a paged cache that are worth a query's attention.  A page's bounds give a bound on the score of any of its tokens:
//   q . k  <=  sum over features of max(q lo, q hi)  =  max(q, 0) . hi + min(q, 0) . lo
// and the bounds of the query heads that share a key head are added, so the weights of hi and lo are sums over those heads and a
// page costs one product of 2 D terms however many heads there are.  Sums are in 64 bits and rounded once to 32: which page is the
// last to be selected does not depend on the order of summation.  (64-bit multiply-adds run at the rate of 32-bit ones here, and
// reading the bounds is what takes the time.)
//
// Two launches: scores as whole numbers in their order (a wavefront's 16-lane group, or 8 or 32 lanes, reads a page's bounds, 16
// bytes a lane), then per sequence and key head the count-th largest by four rounds of histograms of 8 bits, and the pages above
// it in ascending order.
#include "paged_cache_host.h"

namespace iex {
namespace {

struct SelectParams {
  PagedParams cache;
  int group, count, first, last;
  const unsigned short* q;
  long long q_strides[3];
  const unsigned short* bounds;
  unsigned* keys;   // (seqs * kv_heads, table_width)
  int* out;         // (seqs * kv_heads, count)
};

constexpr int kScorePages = 128, kSelectThreads = 512, kSelectKept = 12288;   // pages of a workgroup; ... whose keys fit in LDS

__device__ __forceinline__ int used_pages(const PagedParams& c, int seq) {
  const int length = cached_length(c.lengths[seq], c.table_width, 1 << c.page_shift);
  return (length + (1 << c.page_shift) - 1) >> c.page_shift;
}

template <int CTRL>
__device__ __forceinline__ double dpp_add(double v) {
  const int lo = __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, 0xf, 0xf, true);
  const int hi = __builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, 0xf, 0xf, true);
  return v + __hiloint2double(hi, lo);
}
template <int LANES>
__device__ __forceinline__ double group_sum64(double v) {
  v = dpp_add<0xB1>(v);
  v = dpp_add<0x4E>(v);
  v = dpp_add<0x141>(v);
  if (LANES >= 16) v = dpp_add<0x140>(v);
  if (LANES >= 32) v += __shfl_xor(v, 16);
  return v;
}

template <bool BF16, int D>
__global__ __launch_bounds__(256, D == 256 ? 2 : 4) void page_score_kernel(SelectParams p) {
  constexpr int L = D / 8, P = kWave / L, STEPS = kScorePages / 4 / P;   // lanes of a page, pages of a step
  const PagedParams& c = p.cache;
  const int row = blockIdx.y, seq = row / c.kv_heads, head = row % c.kv_heads;
  const int lane = lane_id(), wave = uniform(threadIdx.x >> 6), used = used_pages(c, seq);
  const int page0 = blockIdx.x * kScorePages + wave * (kScorePages / 4);
  if (page0 >= used) return;
  // where the wavefront's pages lie
  int at = -1;
  if (lane < kScorePages / 4 && page0 + lane < used) at = c.table[(size_t)seq * c.table_row + page0 + lane];
  if ((unsigned)at >= (unsigned)c.pages) at = -1;
  const int d = lane % L * 8;
  u32x4 lo[STEPS], hi[STEPS];
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const int page = __shfl(at, i * P + lane / L);
    lo[i] = hi[i] = u32x4{0u, 0u, 0u, 0u};
    if (page >= 0) {
      const unsigned short* b = p.bounds + ((size_t)page * c.kv_heads + head) * (2 * D) + d;
      lo[i] = *reinterpret_cast<const u32x4*>(b);
      hi[i] = *reinterpret_cast<const u32x4*>(b + D);
    }
  }
  double wl[8], wh[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) wl[j] = wh[j] = 0.0;
  for (int g = 0; g < p.group; ++g) {
    const unsigned short* q = p.q + seq * p.q_strides[0] + (long long)(head * p.group + g) * p.q_strides[1] + d * p.q_strides[2];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float x = f32_of_16<BF16>(q[j * p.q_strides[2]]);
      // (a NaN is in both)
      wl[j] += x > 0.f ? 0.0 : (double)x;
      wh[j] += x < 0.f ? 0.0 : (double)x;
    }
  }
  unsigned* keys = p.keys + (size_t)row * c.table_width;
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float a, b;
      unpack_pair<BF16>(lo[i][j], a, b);
      sum = fma((double)a, wl[2 * j], sum);
      sum = fma((double)b, wl[2 * j + 1], sum);
      unpack_pair<BF16>(hi[i][j], a, b);
      sum = fma((double)a, wh[2 * j], sum);
      sum = fma((double)b, wh[2 * j + 1], sum);
    }
    sum = group_sum64<L>(sum);
    const int number = page0 + i * P + lane / L, page = __shfl(at, i * P + lane / L);
    if (lane % L == 0 && number < used) {
      const bool always = number < p.first || number >= used - p.last;
      keys[number] = page < 0 ? 0u : always ? kSelectAlways : select_key(__float_as_uint((float)sum));
    }
  }
}

// KEPT: the row's keys stay in LDS, else every round reads them again.
template <bool KEPT>
__global__ __launch_bounds__(kSelectThreads) void page_select_kernel(SelectParams p) {
  constexpr int WAVES = kSelectThreads / kWave;
  extern __shared__ unsigned kept[];
  __shared__ unsigned histogram[256];
  __shared__ int chosen[2], totals[2][WAVES];
  const PagedParams& c = p.cache;
  const int row = blockIdx.x, seq = row / c.kv_heads, tid = threadIdx.x, lane = lane_id(), wave = uniform(tid >> 6);
  const int used = used_pages(c, seq);
  const unsigned* keys = p.keys + (size_t)row * c.table_width;
  int* out = p.out + (size_t)row * p.count;
  if (KEPT) {
    for (int i = tid; i < used; i += kSelectThreads) kept[i] = keys[i];
    __syncthreads();
  }
  auto key_of = [&](int i) { return KEPT ? kept[i] : keys[i]; };

  // ---- the count-th largest key ----
  unsigned threshold = 0;
  int need = p.count;   // of the keys that agree with it in the bits found so far, the need-th largest
  if (used > p.count) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += kSelectThreads) histogram[i] = 0;
      __syncthreads();
      for (int i = tid; i < (used + kWave - 1) / kWave * kWave; i += kSelectThreads) {
        const unsigned key = i < used ? key_of(i) : 0u;
        const bool mine = i < used && (shift == 24 || key >> (shift + 8) == threshold >> (shift + 8));
        const int bin = key >> shift & 255;
        // scores of a row share their leading bits: the lanes that agree with the first one are counted at once
        const unsigned long long some = __ballot(mine);
        if (some) {
          const int leader = __ffsll(some) - 1, its = __builtin_amdgcn_readlane(bin, leader);
          const unsigned long long same = __ballot(mine && bin == its);
          if (lane == leader) atomicAdd(&histogram[its], (unsigned)__popcll(same));
          else if (mine && bin != its) atomicAdd(&histogram[bin], 1u);
        }
      }
      __syncthreads();
      if (wave == 0) {   // four bins a lane, from the largest down
        unsigned four[4], mine = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) mine += four[j] = histogram[255 - (lane * 4 + j)];
        unsigned upto = mine;
#pragma unroll
        for (int d = 1; d < kWave; d <<= 1) {
          const unsigned other = __shfl_up(upto, d);
          if (lane >= d) upto += other;
        }
        unsigned above = upto - mine;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (above < (unsigned)need && above + four[j] >= (unsigned)need) chosen[0] = 255 - (lane * 4 + j), chosen[1] = need - (int)above;
          above += four[j];
        }
      }
      __syncthreads();
      threshold |= (unsigned)chosen[0] << shift;
      need = chosen[1];
    }
  }

  // ---- pages above it, and the first `need` that equal it, in ascending order ----
  int written = 0, equal = 0;
  for (int i0 = 0; i0 < used; i0 += kSelectThreads) {
    const int i = i0 + tid;
    const unsigned key = i < used ? key_of(i) : 0u;
    const bool same = key == threshold && key != 0;
    const unsigned long long sames = __ballot(same), below = (1ull << lane) - 1;
    if (lane == 0) totals[0][wave] = __popcll(sames);
    __syncthreads();
    int before = equal;
    for (int w = 0; w < WAVES; ++w) {
      if (w < wave) before += totals[0][w];
      equal += totals[0][w];
    }
    const bool take = key > threshold || (same && before + __popcll(sames & below) < need);
    const unsigned long long takes = __ballot(take);
    if (lane == 0) totals[1][wave] = __popcll(takes);
    __syncthreads();
    int to = written;
    for (int w = 0; w < WAVES; ++w) {
      if (w < wave) to += totals[1][w];
      written += totals[1][w];
    }
    to += __popcll(takes & below);
    if (take && to < p.count) out[to] = i;
  }
  for (int i = written + tid; i < p.count; i += kSelectThreads) out[i] = -1;
}

template <bool BF16>
void launch_scores(const SelectParams& p, int head_dim, hipStream_t s) {
  const dim3 grid(ceil_div(p.cache.table_width, kScorePages), p.cache.seqs * p.cache.kv_heads);
  note_kernel("page_score_kernel<%s, %d>", BF16 ? "bf16" : "f16", head_dim);
  if (head_dim == 64) hipLaunchKernelGGL((page_score_kernel<BF16, 64>), grid, dim3(256), 0, s, p);
  else if (head_dim == 128) hipLaunchKernelGGL((page_score_kernel<BF16, 128>), grid, dim3(256), 0, s, p);
  else hipLaunchKernelGGL((page_score_kernel<BF16, 256>), grid, dim3(256), 0, s, p);
}

}  // namespace
}  // namespace iex

extern "C" size_t iex_select_pages_workspace_bytes(const iex_paged_cache* cache) {
  using namespace iex;
  if (check_paged_cache(cache, "select_pages", false)) return 0;
  return (size_t)cache->seqs * cache->kv_heads * cache->table_width * 4;
}

extern "C" int iex_select_pages(const iex_paged_cache* cache, int heads, const void* q, const long long* q_strides, int count, int first, int last, int* out,
                                void* workspace, size_t workspace_bytes, void* stream) {
  using namespace iex;
  trail_reset();
  if (int rc = check_paged_cache(cache, "select_pages", false)) return rc;
  IEX_REQUIRE(heads >= 0 && (cache->kv_heads == 0 ? heads == 0 : heads % cache->kv_heads == 0), IEX_ERR_BAD_ARGUMENT,
              "select_pages: query heads must be a multiple of key heads (%d, %d)", heads, cache->kv_heads);
  IEX_REQUIRE(count > 0 && first >= 0 && last >= 0 && (long long)first + last <= count, IEX_ERR_BAD_ARGUMENT,
              "select_pages: at least one page, the first and last ones that are always kept among them (count=%d first=%d last=%d)", count, first, last);
  if (cache->seqs == 0 || cache->kv_heads == 0) return 0;
  IEX_REQUIRE((heads == 0 || (q && q_strides)) && out && (cache->bounds || cache->pages == 0), IEX_ERR_BAD_ARGUMENT, "select_pages: null pointer argument");
  IEX_REQUIRE(aligned(q, 2) && aligned(out, 4) && aligned(cache->bounds, 16), IEX_ERR_UNSUPPORTED, "select_pages: operands must be aligned");
  IEX_REQUIRE((long long)cache->seqs * cache->kv_heads < 65536, IEX_ERR_TOO_LARGE, "select_pages: too many sequences or heads");
  const size_t need = iex_select_pages_workspace_bytes(cache);
  IEX_REQUIRE(need == 0 || (workspace && aligned(workspace, 256) && workspace_bytes >= need), IEX_ERR_BAD_ARGUMENT,
              "select_pages: needs a 256-byte aligned workspace of %zu bytes", need);
  SelectParams p{};
  p.cache = paged_params(*cache);
  p.group = heads / cache->kv_heads, p.count = count, p.first = first, p.last = last;
  p.q = static_cast<const unsigned short*>(q), p.bounds = static_cast<const unsigned short*>(cache->bounds);
  for (int i = 0; i < 3; ++i) p.q_strides[i] = heads ? q_strides[i] : 0;
  p.keys = static_cast<unsigned*>(workspace), p.out = out;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (need) {
    if (cache->dtype == IEX_BF16) launch_scores<true>(p, cache->head_dim, s);
    else launch_scores<false>(p, cache->head_dim, s);
    if (int rc = check_hip(hipGetLastError(), "select_pages score launch")) return rc;
  }
  const bool kept = cache->table_width <= kSelectKept;
  note_kernel("page_select_kernel<%s>", kept ? "kept" : "read again");
  const dim3 grid(cache->seqs * cache->kv_heads);
  if (kept) hipLaunchKernelGGL((page_select_kernel<true>), grid, dim3(kSelectThreads), cache->table_width * 4, s, p);
  else hipLaunchKernelGGL((page_select_kernel<false>), grid, dim3(kSelectThreads), 0, s, p);
  return check_hip(hipGetLastError(), "select_pages launch");
}
