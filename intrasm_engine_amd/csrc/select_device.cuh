// The largest of a row of keys (paged_cache.h: whole numbers in the order of scores, 0: not to be taken), in ascending order of their places, by one workgroup.
#pragma once
#include "paged_cache_device.cuh"

namespace iex {

// Four words from place i on of a row of `used`, 0 behind it.  ALIGNED: 16-byte aligned rows.
template <bool ALIGNED>
__device__ __forceinline__ u32x4 four_of(const unsigned* row, int i, int used) {
  typedef u32x4 AnyFour __attribute__((aligned(4)));
  if (i + 4 <= used) {
    if constexpr (ALIGNED) return *reinterpret_cast<const u32x4*>(row + i);
    else return *reinterpret_cast<const AnyFour*>(row + i);
  }
  return u32x4{i < used ? row[i] : 0u, i + 1 < used ? row[i + 1] : 0u, i + 2 < used ? row[i + 2] : 0u, 0u};
}

// The keys of places first .. used - 1 that are above a threshold, and those that equal it as long as fewer than `need` of the row's do before them, in
// ascending order: emit(to, i, payload), to = how many are taken before i.  aboves, equals: how many of the row's keys before `first` are above it, and equal it.
// place(i, before): at every fourth place how many are taken below it.  Returns how many are up to the end.
template <int THREADS, typename KEYS, typename PAYLOADS, typename EMIT, typename PLACE>
__device__ __forceinline__ int take_largest(int first, int used, int count, unsigned threshold, int need, int aboves, int equals, KEYS keys, PAYLOADS payloads, EMIT emit,
                                            PLACE place) {
  constexpr int WAVES = THREADS / kWave, AHEAD = 4, STEP = 4 * kWave;
  __shared__ int totals[2][WAVES];
  const int lane = lane_id(), wave = uniform(threadIdx.x >> 6);
  const int stretch = (used - first + THREADS * 4 - 1) / (THREADS * 4) * STEP, begin = min(used, first + wave * stretch), end = min(used, begin + stretch);
  auto marks = [&](const u32x4& k) {   // (those that equal it, 256 of a step at most) << 16 | those above
    int n = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) n += (k[j] > threshold ? 1 : 0) + (k[j] == threshold && k[j] != 0 ? 1 << 16 : 0);
    return n;
  };
  int above = 0, equal = 0;   // of this lane
  for (int i0 = begin + lane * 4; i0 < end; i0 += AHEAD * STEP) {
    u32x4 k[AHEAD];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) k[a] = i0 + a * STEP < end ? keys(i0 + a * STEP) : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const int n = marks(k[a]);
      above += n & 0xFFFF, equal += n >> 16;
    }
  }
  above = wave_scan(above), equal = wave_scan(equal);
  if (lane == kWave - 1) totals[0][wave] = above, totals[1][wave] = equal;
  __syncthreads();
  int all_above = aboves, all_equal = equals;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    if (w < wave) aboves += totals[0][w], equals += totals[1][w];   // before this wavefront's stretch
    all_above += totals[0][w], all_equal += totals[1][w];
  }
  for (int i0 = begin; i0 < end; i0 += AHEAD * STEP) {
    u32x4 k[AHEAD], what[AHEAD];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const int i = i0 + a * STEP + lane * 4;
      k[a] = what[a] = u32x4{0u, 0u, 0u, 0u};
      if (i < end) k[a] = keys(i), what[a] = payloads(i);
    }
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      if (i0 + a * STEP >= end) break;
      const int i = i0 + a * STEP + lane * 4, mine = marks(k[a]), upto = wave_scan(mine);
      int above_before = aboves + ((upto - mine) & 0xFFFF), equal_before = equals + ((upto - mine) >> 16);
      if (i < end) place(i, above_before + min(equal_before, need));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool more = k[a][j] > threshold, same = k[a][j] == threshold && k[a][j] != 0;
        const int to = above_before + min(equal_before, need);
        if ((more || (same && equal_before < need)) && to < count) emit(to, i + j, what[a][j]);
        above_before += more, equal_before += same;
      }
      const int step = bcast_i(upto, kWave - 1);
      aboves += step & 0xFFFF, equals += step >> 16;
    }
  }
  return min(count, all_above + min(all_equal, need));
}

// The `count` largest of `used` keys (all that are not 0 where there are no more): emit(to, i, payload) for each, to = 0, 1 .. in ascending order of i, by any
// thread; equal keys: the lower places.  keys(i) and payloads(i): four of them from place i on, a multiple of 4; keys behind the row are 0.
// place(i, before): at every fourth place how many were taken below it.  Returns how many were taken.
//
// The count-th largest key by three rounds of histograms, of 11, 11 and 10 bits: the first tells exponents and two bits of the fraction, so that weights
// and scores, which share their leading bits, spread over some bins (lanes that meet in one are added one after the other: 64 clocks where all do).
template <int THREADS, typename KEYS, typename PAYLOADS, typename EMIT, typename PLACE>
__device__ __forceinline__ int select_largest(int used, int count, KEYS keys, PAYLOADS payloads, EMIT emit, PLACE place) {
  constexpr int WAVES = THREADS / kWave, BINS = 2048, EACH = BINS / THREADS, AHEAD = 4;
  static_assert(BINS % THREADS == 0 && EACH >= 1, "bins of a thread");
  __shared__ unsigned histogram[BINS];
  __shared__ int chosen[3], sums[WAVES];
  const int tid = threadIdx.x, lane = lane_id(), wave = uniform(tid >> 6);

  // ---- the count-th largest key ----
  unsigned threshold = 0;
  int need = count;   // of the keys that agree with it in the bits found so far, the need-th largest
  if (used > count) {
    for (int i = tid; i < BINS; i += THREADS) histogram[i] = 0;
    __syncthreads();
#pragma unroll 1
    for (int round = 0; round < 3; ++round) {
      const int shift = round == 0 ? 21 : round == 1 ? 10 : 0, bins = round == 2 ? BINS / 2 : BINS, known = round == 1 ? 21 : 10;
      for (int i0 = tid * 4; i0 < used; i0 += AHEAD * THREADS * 4) {
        u32x4 k[AHEAD];
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) k[a] = keys(i0 + a * THREADS * 4);
#pragma unroll
        for (int a = 0; a < AHEAD; ++a)
#pragma unroll
          for (int j = 0; j < 4; ++j)   // (what is behind the row counts as keys of 0, below all that are taken)
            if (i0 + a * THREADS * 4 < used && (round == 0 || (k[a][j] ^ threshold) >> known == 0)) atomicAdd(&histogram[k[a][j] >> shift & (bins - 1)], 1u);
      }
      __syncthreads();
      // a thread's bins, from the largest down, and how many keys are in the ones above
      unsigned its[EACH], sum = 0;
#pragma unroll
      for (int j = 0; j < EACH; ++j) {
        const int bin = bins - 1 - (tid * EACH + j);
        its[j] = bin >= 0 ? histogram[bin] : 0u;
        if (bin >= 0) histogram[bin] = 0;   // (for the next round)
        sum += its[j];
      }
      const int upto = wave_scan((int)sum);
      if (lane == kWave - 1) sums[wave] = upto;
      __syncthreads();
      unsigned above = (unsigned)upto - sum;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) above += w < wave ? (unsigned)sums[w] : 0u;
#pragma unroll
      for (int j = 0; j < EACH; ++j) {
        if (above < (unsigned)need && above + its[j] >= (unsigned)need)
          chosen[0] = bins - 1 - (tid * EACH + j), chosen[1] = need - (int)above, chosen[2] = above + its[j] == (unsigned)need;
        above += its[j];
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
  return take_largest<THREADS>(0, used, count, threshold, need, 0, 0, keys, payloads, emit, place);
}

}  // namespace iex
