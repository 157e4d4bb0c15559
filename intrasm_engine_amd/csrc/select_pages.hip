// Pages of a paged cache that are worth a query's attention.  A page's bounds give a bound on the score of any of its tokens:
//   q . k  <=  sum over features of max(q lo, q hi)  =  max(q, 0) . hi + min(q, 0) . lo
// and the bounds of the query heads that share a key head are added, so the weights of hi and lo are sums over those heads and a
// page costs one product of 2 D terms however many heads there are.  (An infinite bound under a weight of zero adds nothing, as in the first
// form.)  Sums are in 64 bits and rounded once to 32: another order of summation can change a score only where the sum is within some 2^-45 of it
// from the middle between two 32-bit numbers.  (64-bit multiply-adds run at the rate of 32-bit ones here, and reading the bounds is what takes
// the time.)
//
// Scores are whole numbers in the scores' order (a wavefront's 16-lane group, or 8 or 32 lanes, reads a page's bounds, 16 bytes a
// lane); then the count-th largest by four rounds of histograms of 8 bits, and the pages above it in ascending order.  One workgroup
// does both for a sequence and key head, its scores in LDS, where that keeps the chip busy or the scores are few; else the scores
// come from a launch of their own.
//
// Measured (heads of 128): scores of 8 x 90000 .. 131072 tokens in pages of 32, 8 key heads 25 us = 4.5 TB/s (46 % waiting, 44 % for issue: 64-bit
// conversions take 16 clocks each, which alone would allow 10), selection 10.4; 32 x up to 1024 pages, 8 key heads, in one launch 19 us = 1.9 TB/s,
// 68 % of it waiting (a workgroup a row: the longest set the time).
#include "paged_cache_host.h"

namespace iex {
namespace {

struct SelectParams {
  PagedParams cache;
  int group, count, first, last;
  int per_group;   // pages of a workgroup that only scores
  const unsigned short* q;
  long long q_strides[3];
  const unsigned short* bounds;
  unsigned* keys;   // (seqs * kv_heads, table_width)
  int* out;         // (seqs * kv_heads, count)
};

constexpr int kSelectThreads = 1024, kSelectKept = 12288;   // ... whose pages' scores fit in LDS
constexpr int chunk_of(int head_dim) { return head_dim == 256 ? 16 : 32; }   // pages that a wavefront scores at a time

__device__ __forceinline__ int used_pages(const PagedParams& c, int seq) {
  const int length = cached_length(c.lengths[seq], c.table_width, 1 << c.page_shift);
  return (length + (1 << c.page_shift) - 1) >> c.page_shift;
}

// The value of the lane whose number differs in bit BIT.
template <int BIT>
__device__ __forceinline__ int from_neighbour(int v) {
  if constexpr (BIT == 0) return __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xf, 0xf, true);        // quad_perm [1,0,3,2]
  else if constexpr (BIT == 1) return __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xf, 0xf, true);   // quad_perm [2,3,0,1]
  else if constexpr (BIT == 2) return __builtin_amdgcn_ds_swizzle(v, 0x101F);                    // xor 4
  else if constexpr (BIT == 3) return __builtin_amdgcn_update_dpp(0, v, 0x128, 0xf, 0xf, true);  // row_ror 8
  else return __shfl_xor(v, 1 << BIT);
}
template <int BIT>
__device__ __forceinline__ double from_neighbour(double v) {
  return __hiloint2double(from_neighbour<BIT>(__double2hiint(v)), from_neighbour<BIT>(__double2loint(v)));
}
// COUNT sums over LANES lanes each, at once: in the end lane l has sum number l % COUNT.  (One by one they take four times the additions
// and exchanges.)
template <int COUNT, int LANES, int BIT = 0>
__device__ __forceinline__ double group_sums(double (&v)[COUNT]) {
  if constexpr ((1 << BIT) == LANES) {
    return v[0];
  } else if constexpr ((1 << BIT) < COUNT) {
    const bool odd = lane_id() >> BIT & 1;
    // (the sums left are COUNT >> BIT; every second one goes to the neighbour)
#pragma unroll
    for (int k = 0; k < (COUNT >> BIT) / 2; ++k) {
      const double mine = odd ? v[2 * k + 1] : v[2 * k], other = odd ? v[2 * k] : v[2 * k + 1];
      v[k] = mine + from_neighbour<BIT>(other);
    }
    return group_sums<COUNT, LANES, BIT + 1>(v);
  } else {
    v[0] += from_neighbour<BIT>(v[0]);
    return group_sums<COUNT, LANES, BIT + 1>(v);
  }
}

// The weights of smallest and largest keys for a sequence and key head, into LDS (by all threads; a barrier follows).
template <bool BF16, int D>
__device__ __forceinline__ void page_weights(const SelectParams& p, int seq, int head, double (&weights)[2 * D]) {
  for (int d = threadIdx.x; d < D; d += blockDim.x) {
    double low = 0.0, high = 0.0;
    const unsigned short* q = p.q + seq * p.q_strides[0] + (long long)head * p.group * p.q_strides[1] + d * p.q_strides[2];
    for (int g0 = 0; g0 < p.group; g0 += 8) {   // (eight loads at a time: one after the other they take a microsecond each)
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = f32_of_16<BF16>(q[min(g0 + i, p.group - 1) * p.q_strides[1]]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (g0 + i >= p.group) break;
        low += x[i] > 0.f ? 0.0 : (double)x[i];   // (a NaN is in both)
        high += x[i] < 0.f ? 0.0 : (double)x[i];
      }
    }
    weights[d] = low, weights[D + d] = high;
  }
}

// The scores of chunks of a row's pages from page0 on, every `step` pages, to keys[].  `all`: there are no more pages than are
// wanted, so each that exists is.
template <bool BF16, int D>
__device__ __forceinline__ void score_pages(const SelectParams& p, int seq, int head, int used, int page0, int step, int end, bool all, const double (&weights)[2 * D],
                                            unsigned* keys) {
  constexpr int L = D / 8, P = kWave / L, CHUNK = chunk_of(D), STEPS = CHUNK / P;   // lanes of a page, pages of a step
  const PagedParams& c = p.cache;
  const int lane = lane_id(), d = lane % L * 8;
  const int* table = c.table + (size_t)seq * c.table_row;
  auto find = [&](int first) {   // where a chunk's pages lie, one a lane
    const int number = first + lane;
    const int at = lane < CHUNK && number < used ? table[number] : -1;
    return (unsigned)at < (unsigned)c.pages ? at : -1;
  };
  if (page0 >= end) return;
  int at = find(page0);
  if (all) {
    for (; page0 < end; page0 += step) {
      if (lane < CHUNK && page0 + lane < used) keys[page0 + lane] = at < 0 ? 0u : kSelectAlways;
      if (page0 + step < end) at = find(page0 + step);
    }
    return;
  }
  const int first = page0;
  bool some_nan = false;
  double wl[8], wh[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) wl[j] = weights[d + j], wh[j] = weights[D + d + j];
  for (; page0 < end; page0 += step) {
    u32x4 lo[STEPS], hi[STEPS];
    const int instead = max(0, bcast_i(at, 0));
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {   // (in the place of a page that is not there: the chunk's first)
      const int page = __shfl(at, i * P + lane / L);
      const unsigned short* b = p.bounds + ((size_t)(page < 0 ? instead : page) * c.kv_heads + head) * (2 * D) + d;
      lo[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(b));
      hi[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(b + D));
    }
    const int next = page0 + step < end ? find(page0 + step) : -1;
    double sums[STEPS];
#pragma unroll
    for (int i = 0; i < STEPS; ++i) sums[i] = 0.0;
#pragma unroll
    for (int j = 0; j < 4; ++j)   // (the steps side by side: one sum is a chain)
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        float a, b;
        unpack_pair<BF16>(lo[i][j], a, b);
        sums[i] = fma((double)a, wl[2 * j], sums[i]);
        sums[i] = fma((double)b, wl[2 * j + 1], sums[i]);
        unpack_pair<BF16>(hi[i][j], a, b);
        sums[i] = fma((double)a, wh[2 * j], sums[i]);
        sums[i] = fma((double)b, wh[2 * j + 1], sums[i]);
      }
    const double sum = group_sums<STEPS, L>(sums);
    some_nan |= __ballot(sum != sum) != 0;
    const int in_chunk = lane % STEPS * P + lane / L, number = page0 + in_chunk, page = __shfl(at, in_chunk);
    const bool always = number < p.first || number >= used - p.last;
    if (lane % L < STEPS && number < used) keys[number] = page < 0 ? 0u : always ? kSelectAlways : select_key(__float_as_uint((float)sum));
    at = next;
  }
  if (!some_nan) return;
  // (rare) NaN, or an infinite bound under a weight of zero, which adds nothing: those pages again, one by one, with a look at every term.
  // In the loop above it costs more registers: with the attention 32 x up to 1024 pages 72.3 us (here 70.5), 8 x 90000 .. 131072 tokens 61.3 (60.8;
  // without it 71.0 and 59.6).
  __threadfence_block();
  for (page0 = first; page0 < end; page0 += step) {
    const int number = page0 + lane;
    for (unsigned long long left = __ballot(lane < CHUNK && number < used && keys[number] == kSelectNaN); left; left &= left - 1) {
      const int again = page0 + __ffsll(left) - 1;
      const unsigned short* b = p.bounds + ((size_t)table[again] * c.kv_heads + head) * (2 * D);
      double sum = 0.0;
      for (int i = lane; i < 2 * D; i += kWave) {
        const float x = f32_of_16<BF16>(b[i]);
        if (weights[i] != 0.0 || fabsf(x) != INFINITY) sum = fma((double)x, weights[i], sum);
      }
#pragma unroll
      for (int bit = 1; bit < kWave; bit *= 2) sum += __shfl_xor(sum, bit);
      if (lane == 0) keys[again] = select_key(__float_as_uint((float)sum));
    }
  }
}

template <bool BF16, int D>
__global__ __launch_bounds__(256, D == 256 ? 2 : 4) void page_score_kernel(SelectParams p) {
  __shared__ double weights[2 * D];
  const PagedParams& c = p.cache;
  const int row = blockIdx.y, seq = row / c.kv_heads, head = row % c.kv_heads, wave = uniform(threadIdx.x >> 6);
  const int used = used_pages(c, seq), first = blockIdx.x * p.per_group, end = min(used, first + p.per_group);
  if (first >= end) return;
  page_weights<BF16, D>(p, seq, head, weights);
  __syncthreads();
  score_pages<BF16, D>(p, seq, head, used, first + wave * chunk_of(D), 4 * chunk_of(D), end, used <= p.count || c.pages == 0, weights, p.keys + (size_t)row * c.table_width);
}

// KEPT: the row's keys stay in LDS, else every round reads them again.  SCORED: they are in p.keys, else they are worked out here
// (from D features of 16 bits; KEPT only).
template <bool KEPT, bool SCORED, bool BF16, int D>
__global__ __launch_bounds__(kSelectThreads) void page_select_kernel(SelectParams p) {
  constexpr int WAVES = kSelectThreads / kWave;
  extern __shared__ unsigned kept[];
  __shared__ double weights[SCORED ? 2 : 2 * D];
  __shared__ unsigned histogram[256];
  __shared__ int chosen[3], totals[2][WAVES];
  const PagedParams& c = p.cache;
  const int row = blockIdx.x, seq = row / c.kv_heads, tid = threadIdx.x, lane = lane_id(), wave = uniform(tid >> 6);
  const int used = used_pages(c, seq);
  const unsigned* keys = SCORED ? p.keys + (size_t)row * c.table_width : nullptr;
  int* out = p.out + (size_t)row * p.count;
  if constexpr (!SCORED) {
    page_weights<BF16, D>(p, seq, row % c.kv_heads, weights);
    __syncthreads();
    score_pages<BF16, D>(p, seq, row % c.kv_heads, used, wave * chunk_of(D), WAVES * chunk_of(D), used, used <= p.count || c.pages == 0, weights, kept);
  } else if (KEPT) {
    for (int i = tid; i < used; i += kSelectThreads) kept[i] = keys[i];
  }
  __syncthreads();
  auto key_of = [&](int i) { return KEPT ? kept[i] : keys[i]; };

  // ---- the count-th largest key ----
  unsigned threshold = 0;
  int need = p.count;   // of the keys that agree with it in the bits found so far, the need-th largest
  if (used > p.count) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) histogram[tid] = 0;
      __syncthreads();
      for (int i0 = wave * kWave; i0 < used; i0 += kSelectThreads) {
        const int i = i0 + lane;
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
        unsigned above = (unsigned)wave_scan((int)mine) - mine;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (above < (unsigned)need && above + four[j] >= (unsigned)need)
            chosen[0] = 255 - (lane * 4 + j), chosen[1] = need - (int)above, chosen[2] = above + four[j] == (unsigned)need;
          above += four[j];
        }
      }
      __syncthreads();
      threshold |= (unsigned)chosen[0] << shift;
      need = chosen[1];
      if (chosen[2] && threshold != 0) {   // all that agree so far are wanted: whatever follows (and nothing below)
        --threshold, need = 0;
        break;
      }
    }
  }

  // ---- pages above it, and the first `need` that equal it, in ascending order: a wavefront has a stretch of pages ----
  const int stretch = (used + kSelectThreads - 1) / kSelectThreads * kWave, begin = min(used, wave * stretch), end = min(used, begin + stretch);
  int above = 0, equal = 0;
  for (int i0 = begin; i0 < end; i0 += kWave) {
    const unsigned key = i0 + lane < end ? key_of(i0 + lane) : 0u;
    above += __popcll(__ballot(key > threshold));
    equal += __popcll(__ballot(key == threshold && key != 0));
  }
  if (lane == 0) totals[0][wave] = above, totals[1][wave] = equal;
  __syncthreads();
  int written = 0, equals = 0, all = 0;   // before this wavefront's stretch; all pages that are taken
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    const int taken = min(totals[1][w], max(0, need - equals));
    if (w < wave) written += totals[0][w] + taken;
    all += totals[0][w] + taken;
    equals += totals[1][w];
  }
  equals = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) equals += w < wave ? totals[1][w] : 0;
  for (int i0 = begin; i0 < end; i0 += kWave) {
    const unsigned key = i0 + lane < end ? key_of(i0 + lane) : 0u;
    const bool same = key == threshold && key != 0;
    const unsigned long long sames = __ballot(same), below = (1ull << lane) - 1;
    const bool take = key > threshold || (same && equals + __popcll(sames & below) < need);
    const unsigned long long takes = __ballot(take);
    const int to = written + __popcll(takes & below);
    if (take && to < p.count) out[to] = i0 + lane;
    written += __popcll(takes), equals += __popcll(sames);
  }
  for (int i = all + tid; i < p.count; i += kSelectThreads) out[i] = -1;
}

// One launch where the scores are few (a row's pages on one CU: 256 9.1 us against 10.3, 512 11.1 against 9.9, 2048 31 against 13) or rows
// enough for the chip (256 of 1024 28.1 against 31.8, 128 of 1024 21.3 against 20.1).
bool one_launch(const iex_paged_cache& c) {
  return c.table_width <= kSelectKept && (c.table_width <= 256 || (long long)c.seqs * c.kv_heads >= 256);
}

template <bool BF16, int D>
void launch_forms(const SelectParams& p, bool once, hipStream_t s) {
  const int rows = p.cache.seqs * p.cache.kv_heads, width = p.cache.table_width;
  if (once) {
    note_kernel("page_select_kernel<%s, %d>", BF16 ? "bf16" : "f16", D);
    hipLaunchKernelGGL((page_select_kernel<true, false, BF16, D>), dim3(rows), dim3(kSelectThreads), width * 4, s, p);
    return;
  }
  note_kernel("page_score_kernel<%s, %d>", BF16 ? "bf16" : "f16", D);
  // a chunk for each of four wavefronts, two where there are workgroups enough (the weights are made once a workgroup): 8 rows of 2048 pages
  // 13.3 us by one, 15.7 by two; 32 of 8192 42.2, 40.5, by four 41.2
  SelectParams scores = p;
  const long long chunks = (long long)ceil_div(width, 4 * chunk_of(D)) * rows;
  scores.per_group = 4 * chunk_of(D) * (chunks >= 1024 ? 2 : 1);
  hipLaunchKernelGGL((page_score_kernel<BF16, D>), dim3(ceil_div(width, scores.per_group), rows), dim3(256), 0, s, scores);
  if (width <= kSelectKept) {
    note_kernel("page_select_kernel<kept>");
    hipLaunchKernelGGL((page_select_kernel<true, true, true, 64>), dim3(rows), dim3(kSelectThreads), width * 4, s, p);
  } else {
    note_kernel("page_select_kernel<read again>");
    hipLaunchKernelGGL((page_select_kernel<false, true, true, 64>), dim3(rows), dim3(kSelectThreads), 0, s, p);
  }
}

template <bool BF16>
void launch_dim(const SelectParams& p, int head_dim, bool once, hipStream_t s) {
  if (head_dim == 64) launch_forms<BF16, 64>(p, once, s);
  else if (head_dim == 128) launch_forms<BF16, 128>(p, once, s);
  else launch_forms<BF16, 256>(p, once, s);
}

}  // namespace
}  // namespace iex

extern "C" size_t iex_select_pages_workspace_bytes(const iex_paged_cache* cache) {
  using namespace iex;
  if (check_paged_cache(cache, "select_pages", false)) return 0;
  return one_launch(*cache) ? 0 : (size_t)cache->seqs * cache->kv_heads * cache->table_width * 4;
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
  // (2^32 threads a launch; scores in a launch of their own have a row in the grid's second dimension)
  IEX_REQUIRE((long long)cache->seqs * cache->kv_heads < (one_launch(*cache) ? 1 << 22 : 65536), IEX_ERR_TOO_LARGE, "select_pages: too many sequences or heads");
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
  if (cache->dtype == IEX_BF16) launch_dim<true>(p, cache->head_dim, one_launch(*cache), s);
  else launch_dim<false>(p, cache->head_dim, one_launch(*cache), s);
  return check_hip(hipGetLastError(), "select_pages launch");
}
