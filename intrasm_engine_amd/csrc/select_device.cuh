// The largest of a row of keys (paged_cache.h: whole numbers in the order of scores, 0: not to be taken), in ascending order of their places, by one workgroup.
#pragma once
#include "paged_cache_device.cuh"

namespace iex {

// The `count` largest of `used` keys (all that are not 0 where there are no more): emit(to, i) for each, to = 0, 1 .. in ascending order of i, by any
// thread; equal keys: the lower places.  window(i0, before): before each 64 places from i0 on how many were taken below them (all lanes of a wavefront, not
// every workgroup's).  By four rounds of histograms of 8 bits.  Returns how many were taken.
template <int THREADS, typename KEY, typename EMIT, typename WINDOW>
__device__ __forceinline__ int select_largest(int used, int count, KEY key_of, EMIT emit, WINDOW window) {
  constexpr int WAVES = THREADS / kWave;
  __shared__ unsigned histogram[256];
  __shared__ int chosen[3], totals[2][WAVES];
  const int tid = threadIdx.x, lane = lane_id(), wave = uniform(tid >> 6);

  // ---- the count-th largest key ----
  unsigned threshold = 0;
  int need = count;   // of the keys that agree with it in the bits found so far, the need-th largest
  if (used > count) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) histogram[tid] = 0;
      __syncthreads();
      for (int i0 = wave * kWave; i0 < used; i0 += THREADS) {
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

  // ---- what is above it, and the first `need` that equal it, in ascending order: a wavefront has a stretch ----
  const int stretch = (used + THREADS - 1) / THREADS * kWave, begin = min(used, wave * stretch), end = min(used, begin + stretch);
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
    window(i0, min(written, count));
    const unsigned key = i0 + lane < end ? key_of(i0 + lane) : 0u;
    const bool same = key == threshold && key != 0;
    const unsigned long long sames = __ballot(same), below = (1ull << lane) - 1;
    const bool take = key > threshold || (same && equals + __popcll(sames & below) < need);
    const unsigned long long takes = __ballot(take);
    const int to = written + __popcll(takes & below);
    if (take && to < count) emit(to, i0 + lane);
    written += __popcll(takes), equals += __popcll(sames);
  }
  return all;
}

}  // namespace iex
