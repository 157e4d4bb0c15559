// Tokens of a paged cache that got least attention leave it.  Of a sequence of n > keep tokens every key head keeps the first `first`, the last `recent` and,
// of those between, the ones with the largest accumulated weight (paged_account.hip), the earlier of two that are equal; they move, in order, to places
// 0 .. keep - 1 of the sequence's own pages, their weights with them, and the sequence has `keep` tokens.
//
// First the list of kept tokens, ascending: by a workgroup a sequence and key head whose keys are in LDS (select_device.cuh), for tables of more than 32768
// tokens by slices of 8192, in a launch for each eight bits of the keys and one that takes what is above.
// Then a launch that moves rows, in place: chunk c of a list, up to `chunk` tokens, reads rows that others may be about to write.  The i-th kept token is
// at place i or behind it, so what chunk c writes, places c * chunk and on, is only ever read by itself and by chunks before it (the list's stretch
// with tokens there ends before its own); all of a chunk's rows are in registers before its first write, and it writes when the chunks before it that
// read there, two at most, have said that theirs are too.  Chunks are drawn by ticket: the one that is waited for has been drawn before, by a workgroup that is
// running and that waits for nobody before it has read, so every wait ends.  It is bounded all the same, to about a second, for calls that share a workspace at
// the same time, which they must not: a chunk that gives up leaves NaN in the places that it should have written, and -2 in the list.
//
// What bounds it: memory, kept rows read and written once: 64 sequences of 1500 .. 4224 tokens to 2048, 8 key heads of 128 in 16 bits 150 us = 5.0 TB/s,
// selection 17; 131071 tokens to 32768, every fourth row of 256 bytes, 67 us = 4.1 TB/s, selection 32 in five launches (by one workgroup a row, whose CU reads
// the weights again in every round, 143); 700 tokens to 512, 32 key heads 6.4, selection 6.9.  The 64 sequences with weights spread evenly 134 us, in e4m3
// 66; bounds of their pages another 126, e4m3 86 (evict_bounds_kernel).
#include "paged_cache_host.h"
#include "select_device.cuh"

namespace iex {
namespace {

struct EvictParams {
  PagedParams cache;
  int keep, first, recent, chunks;   // chunks of a list
  int* lengths;
  float* weights;      // (seqs, kv_heads, tokens of a table)
  int* kept;           // (seqs, kv_heads, keep)
  unsigned short* bounds;
  // the workspace; rows are a sequence's key heads
  int* tokens;         // (rows) tokens of a row that is cut, else 0
  int* tickets;        // (rows) chunks drawn
  int* flags;          // (rows, chunks) 1: read
  int* before;         // (rows, chunks + 1) how many tokens before place i * chunk are kept
  float* kept_weights; // (rows, keep)
  unsigned* histograms;   // slices: two of (rows, slices, 256)
  int4* found;            // ... (rows, slices) what of the threshold is known, how many that agree with it are wanted, how many before the slice are above it
  int slices;
  int tries;              // of a wait
};

constexpr int kEvictThreads = 1024, kEvictKept = 32768;   // ... whose weights fit in LDS
constexpr int kEvictSlice = 8192;                         // tokens
constexpr int kEvictTries = 1 << 20;                      // of a wait: about a second

// Four words from place i on of a 16-byte aligned row of `used`, 0 behind it.
__device__ __forceinline__ u32x4 four_of(const unsigned* row, int i, int used) {
  if (i + 4 <= used) return *reinterpret_cast<const u32x4*>(row + i);
  return u32x4{i < used ? row[i] : 0u, i + 1 < used ? row[i + 1] : 0u, i + 2 < used ? row[i + 2] : 0u, 0u};
}

// The keys of a slice, places first .. used - 1 of a row, that are above a threshold, and those that equal it as long as fewer than `need` of the row's do
// before them, in ascending order: emit(to, i, payload), to = how many are taken before i.  aboves, equals: how many of the row's keys before `first` are above
// it, and equal it.  place(i, before): at every fourth place how many are taken below it.  A wavefront has a stretch of 64 x 4 x STEPS places.
template <int THREADS, int STEPS, typename KEYS, typename PAYLOADS, typename EMIT, typename PLACE>
__device__ __forceinline__ void take_largest(int first, int used, int count, unsigned threshold, int need, int aboves, int equals, KEYS keys, PAYLOADS payloads, EMIT emit,
                                             PLACE place) {
  constexpr int WAVES = THREADS / kWave, STEP = 4 * kWave;
  __shared__ int totals[2][WAVES];
  const int lane = lane_id(), wave = uniform(threadIdx.x >> 6), begin = first + wave * (STEPS * STEP);
  u32x4 k[STEPS], what[STEPS];
#pragma unroll
  for (int a = 0; a < STEPS; ++a) k[a] = keys(begin + a * STEP + lane * 4);   // (0 behind the row)
#pragma unroll
  for (int a = 0; a < STEPS; ++a) what[a] = payloads(begin + a * STEP + lane * 4);
  auto marks = [&](const u32x4& key) {   // (those that equal it, 256 of a step at most) << 16 | those above
    int n = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) n += (key[j] > threshold ? 1 : 0) + (key[j] == threshold && key[j] != 0 ? 1 << 16 : 0);
    return n;
  };
  int mine[STEPS], upto[STEPS], above = 0, equal = 0;   // a step's own marks, with the lanes before; the wavefront's
#pragma unroll
  for (int a = 0; a < STEPS; ++a) {
    mine[a] = marks(k[a]), upto[a] = wave_scan(mine[a]);
    const int step = bcast_i(upto[a], kWave - 1);
    above += step & 0xFFFF, equal += step >> 16;
  }
  if (lane == 0) totals[0][wave] = above, totals[1][wave] = equal;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WAVES; ++w)
    if (w < wave) aboves += totals[0][w], equals += totals[1][w];
#pragma unroll
  for (int a = 0; a < STEPS; ++a) {
    const int i = begin + a * STEP + lane * 4;
    int above_before = aboves + ((upto[a] - mine[a]) & 0xFFFF), equal_before = equals + ((upto[a] - mine[a]) >> 16);
    if (i < used) place(i, above_before + min(equal_before, need));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool more = k[a][j] > threshold, same = k[a][j] == threshold && k[a][j] != 0;
      const int to = above_before + min(equal_before, need);
      if ((more || (same && equal_before < need)) && to < count) emit(to, i + j, what[a][j]);
      above_before += more, equal_before += same;
    }
    const int step = bcast_i(upto[a], kWave - 1);
    aboves += step & 0xFFFF, equals += step >> 16;
  }
}

// Whether a row is to be cut.  One that is not gets its list here (all of a sequence that is short enough, or nothing: a sequence with pages given back has no
// place for what it keeps), by the workgroups that are `one`; all of a row's workgroups see the same.
template <int THREADS>
__device__ __forceinline__ bool evict_begin(const EvictParams& p, int row, int length, bool one) {
  const PagedParams& c = p.cache;
  const int seq = row / c.kv_heads, tid = threadIdx.x;
  bool gone = false;
  if (length > p.keep)
    for (int i = tid; i << c.page_shift < length; i += THREADS) gone |= (unsigned)c.table[(size_t)seq * c.table_row + i] >= (unsigned)c.pages;
  const bool cut = !__syncthreads_or(gone) && length > p.keep;
  if (!one) return cut;
  if (!cut) {
    int* const kept = p.kept + (size_t)row * p.keep;
    for (int i = tid; i < p.keep; i += THREADS) kept[i] = length <= p.keep && i < length ? i : -1;
  } else {
    for (int i = tid; i < p.chunks; i += THREADS) p.flags[(size_t)row * p.chunks + i] = 0;
  }
  if (tid == 0) p.tokens[row] = cut ? length : 0, p.tickets[row] = 0;
  return cut;
}

// Keys of a row's weights, and what becomes of those that are taken.
struct EvictRow {
  const EvictParams& p;
  int length, chunk_shift;
  const unsigned* weights;
  int *kept, *before;
  unsigned* moved;
  __device__ __forceinline__ EvictRow(const EvictParams& params, int row, int tokens, int shift) : p(params), length(tokens), chunk_shift(shift) {
    weights = reinterpret_cast<const unsigned*>(p.weights) + (size_t)row * ((size_t)p.cache.table_width << p.cache.page_shift);
    kept = p.kept + (size_t)row * p.keep, before = p.before + (size_t)row * (p.chunks + 1);
    moved = reinterpret_cast<unsigned*>(p.kept_weights) + (size_t)row * p.keep;
  }
  __device__ __forceinline__ u32x4 weights_at(int i) const { return four_of(weights, i, length); }
  __device__ __forceinline__ u32x4 keys_at(int i) const {
    u32x4 four = weights_at(i);
#pragma unroll
    for (int j = 0; j < 4; ++j) four[j] = i + j >= length ? 0u : i + j < p.first || i + j >= length - p.recent ? kSelectAlways : select_key(four[j]);
    return four;
  }
  __device__ __forceinline__ void take(int to, int i, unsigned weight) const { kept[to] = i, moved[to] = weight; }
  __device__ __forceinline__ void place(int i, int taken) const {
    if ((i & ((1 << chunk_shift) - 1)) == 0 && i >> chunk_shift <= p.chunks) before[i >> chunk_shift] = taken;
  }
};

__device__ __forceinline__ int evict_length(const PagedParams& c, int row) { return cached_length(c.lengths[row / c.kv_heads], c.table_width, 1 << c.page_shift); }

template <int THREADS>
__global__ __launch_bounds__(THREADS) void evict_select_kernel(EvictParams p, int chunk_shift) {
  extern __shared__ __align__(16) unsigned keys[];
  const int row = blockIdx.x, length = evict_length(p.cache, row);
  const EvictRow its(p, row, length, chunk_shift);
  if (length > p.keep) {   // (beside the look at the pages)
#pragma unroll 4
    for (int i = threadIdx.x * 4; i < length; i += THREADS * 4) *reinterpret_cast<u32x4*>(keys + i) = its.keys_at(i);   // (a table's tokens are a multiple of 16)
  }
  if (!evict_begin<THREADS>(p, row, length, true)) return;
  select_largest<THREADS>(
      length, p.keep, [&](int i) { return keys[i]; }, [&](int to, int i) { its.take(to, i, its.weights[i]); },
      [&](int i, int taken) {
        if (lane_id() == 0) its.place(i, taken);
      });
}

// Slices: launch STAGE 0 .. 3 counts the keys that agree with what is known of the threshold by their next eight bits, a histogram a slice; the next
// launch's workgroups each add up all of their row's histograms and know eight bits more, how many of those that agree are wanted, and how many keys
// in slices before theirs are above the threshold.  Launch 4 takes what is above it.  Nobody waits for another workgroup, and no sum depends on an order.
template <int STAGE>
__global__ __launch_bounds__(kEvictThreads) void evict_slice_kernel(EvictParams p, int chunk_shift) {
  __shared__ unsigned histogram[256], total[4][256], earlier[4][256];
  __shared__ int chosen[4];   // bin, still wanted, above it in earlier slices, equal to it there
  const PagedParams& c = p.cache;
  const int row = blockIdx.x / p.slices, slice = blockIdx.x % p.slices, tid = threadIdx.x, lane = lane_id();
  int length;
  if constexpr (STAGE == 0) {
    length = evict_length(c, row);
    if (slice != 0 && slice * kEvictSlice >= length) return;
    if (!evict_begin<kEvictThreads>(p, row, length, slice == 0)) return;
  } else {
    length = p.tokens[row];
    if (slice * kEvictSlice >= length) return;   // (0 where a row is not cut)
  }
  const EvictRow its(p, row, length, chunk_shift);
  const int first = slice * kEvictSlice, used = min(length, first + kEvictSlice), slices = (length + kEvictSlice - 1) / kEvictSlice;
  const size_t all = (size_t)c.seqs * c.kv_heads * p.slices;   // histograms of a launch
  int4 found{0, p.keep, 0, 0};
  if constexpr (STAGE > 0) {
    if (STAGE > 1) found = p.found[(size_t)row * p.slices + slice];
    const unsigned* from = p.histograms + ((STAGE - 1) % 2 * all + (size_t)row * p.slices) * 256;
    unsigned sum = 0, mine = 0;
    for (int s = tid >> 8; s < slices; s += 4) {
      const unsigned n = from[s * 256 + (tid & 255)];
      sum += n, mine += s < slice ? n : 0u;
    }
    total[tid >> 8][tid & 255] = sum, earlier[tid >> 8][tid & 255] = mine;
    __syncthreads();
    if (tid < kWave) {   // four bins a lane, from the largest down
      unsigned four[4], before[4], in_lane = 0, before_in_lane = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int bin = 255 - (lane * 4 + j);
        four[j] = total[0][bin] + total[1][bin] + total[2][bin] + total[3][bin];
        before[j] = earlier[0][bin] + earlier[1][bin] + earlier[2][bin] + earlier[3][bin];
        in_lane += four[j], before_in_lane += before[j];
      }
      unsigned above = (unsigned)wave_scan((int)in_lane) - in_lane, above_before = (unsigned)wave_scan((int)before_in_lane) - before_in_lane;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (above < (unsigned)found.y && above + four[j] >= (unsigned)found.y)
          chosen[0] = 255 - (lane * 4 + j), chosen[1] = found.y - (int)above, chosen[2] = (int)above_before, chosen[3] = (int)before[j];
        above += four[j], above_before += before[j];
      }
    }
    __syncthreads();
    found.x |= chosen[0] << (32 - 8 * STAGE), found.y = chosen[1], found.z += chosen[2], found.w = chosen[3];
    if (STAGE < 4 && tid == 0) p.found[(size_t)row * p.slices + slice] = found;
  }
  if constexpr (STAGE < 4) {
    constexpr int shift = 24 - 8 * STAGE;
    for (int i = tid; i < 256; i += kEvictThreads) histogram[i] = 0;
    __syncthreads();
    u32x4 k[kEvictSlice / (kEvictThreads * 4)];
#pragma unroll
    for (int a = 0; a < kEvictSlice / (kEvictThreads * 4); ++a) k[a] = its.keys_at(first + (a * kEvictThreads + tid) * 4);
#pragma unroll
    for (int a = 0; a < kEvictSlice / (kEvictThreads * 4); ++a)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        bool counts = first + (a * kEvictThreads + tid) * 4 + j < used;
        if constexpr (STAGE > 0) counts = counts && (k[a][j] ^ (unsigned)found.x) >> (shift + 8) == 0;
        if (counts) atomicAdd(&histogram[k[a][j] >> shift & 255], 1u);
      }
    __syncthreads();
    unsigned* to = p.histograms + (STAGE % 2 * all + (size_t)row * p.slices + slice) * 256;
    if (tid < 256) to[tid] = histogram[tid];
  } else {
    take_largest<kEvictThreads, kEvictSlice / (kEvictThreads * 4)>(
        first, used, p.keep, (unsigned)found.x, found.y, found.z, found.w, [&](int i) { return its.keys_at(i); }, [&](int i) { return its.weights_at(i); },
        [&](int to, int i, unsigned weight) { its.take(to, i, weight); }, [&](int i, int taken) { its.place(i, taken); });
  }
}

// Tokens of a chunk: sixteen 16-byte loads of 256 threads, of keys and values (131071 -> 32768 tokens, 8 key heads of 128: 66 us, by eight loads 80), and no
// more than there are threads.
constexpr int evict_chunk(int row_bytes) { return 16 * 256 * 16 / (2 * row_bytes) > 256 ? 256 : 16 * 256 * 16 / (2 * row_bytes); }

// ROW: bytes of a token's key or value of one head.
template <int ROW, bool E8>
__global__ __launch_bounds__(256) void evict_move_kernel(EvictParams p) {
  constexpr int T = evict_chunk(ROW), LANES = ROW / 16, LOADS = T * LANES / 256;   // tokens; 16-byte pieces of a row; loads of a thread, of keys and of values
  const PagedParams& c = p.cache;
  const int rows = c.seqs * c.kv_heads, row = blockIdx.x % rows, seq = row / c.kv_heads, head = row % c.kv_heads, tid = threadIdx.x;
  const int length = p.tokens[row];
  if (length == 0) return;
  __shared__ int drawn;
  __shared__ int from[T], to[T];   // rows before a token's in the cache, page by page: page << page_shift | slot
  if (tid == 0) drawn = atomicAdd(p.tickets + row, 1);
  __syncthreads();
  const int chunk = drawn, first = chunk * T, count = min(T, p.keep - first);
  if ((unsigned)chunk >= (unsigned)p.chunks) return;
  const int* const kept = p.kept + (size_t)row * p.keep;
  float* const weights = p.weights + (size_t)row * ((size_t)c.table_width << c.page_shift);
  // the weights, which nobody reads here: those of the chunk's tokens, and this chunk's share of the zeros behind the kept ones
  for (int i = tid; i < count; i += 256) weights[first + i] = p.kept_weights[(size_t)row * p.keep + first + i];
  const int share = (length - p.keep + p.chunks - 1) / p.chunks;
  for (int i = p.keep + chunk * share + tid; i < min(length, p.keep + (chunk + 1) * share); i += 256) weights[i] = 0.f;
  if (head == 0 && chunk == 0 && tid == 0) p.lengths[seq] = p.keep;
  if (kept[first + count - 1] == first + count - 1) return;   // all of them are where they belong

  const int* const table = c.table + (size_t)seq * c.table_row;
  for (int i = tid; i < T; i += 256) {   // (behind the last one: that one again)
    const int t = first + min(i, count - 1), source = kept[t];
    from[i] = table[source >> c.page_shift] << c.page_shift | (source & ((1 << c.page_shift) - 1));
    to[i] = table[t >> c.page_shift] << c.page_shift | (t & ((1 << c.page_shift) - 1));
  }
  __syncthreads();
  auto row_at = [&](int place, long long page_stride) {   // elements are bytes where E8, else two
    const int page = place >> c.page_shift, slot = place & ((1 << c.page_shift) - 1);
    return (page * page_stride) * (E8 ? 1 : 2) + ((long long)(head << c.page_shift) + slot) * ROW;
  };
  auto exponent_at = [&](int place) {
    const int page = place >> c.page_shift, slot = place & ((1 << c.page_shift) - 1);
    return (((size_t)page * c.kv_heads + head) << c.page_shift) + slot;
  };
  unsigned char* const keys = static_cast<unsigned char*>(const_cast<void*>(c.keys));
  unsigned char* const values = static_cast<unsigned char*>(const_cast<void*>(c.values));
  unsigned char* const key_exponents = const_cast<unsigned char*>(c.key_exponents);
  unsigned char* const value_exponents = const_cast<unsigned char*>(c.value_exponents);
  const int piece = tid % LANES * 16, line = tid / LANES;
  u32x4 k[LOADS], v[LOADS];
  unsigned char ke = 0, ve = 0;
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int place = from[line + i * (256 / LANES)];
    k[i] = *reinterpret_cast<const u32x4*>(keys + row_at(place, c.key_page) + piece);
    v[i] = *reinterpret_cast<const u32x4*>(values + row_at(place, c.value_page) + piece);
  }
  if constexpr (E8) {
    static_assert(T <= 256, "a thread has a token's exponents");
    if (tid < T) ke = key_exponents[exponent_at(from[tid])], ve = value_exponents[exponent_at(from[tid])];
  }
  const EvictReaders readers = evict_readers(chunk, T, length, p.before + (size_t)row * (p.chunks + 1));
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  int* const flags = p.flags + (size_t)row * p.chunks;
  if (tid == 0) __hip_atomic_store(flags + chunk, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  bool read = true;
  if (tid < readers.count) {
    read = false;
    for (int tries = 0; tries < p.tries && !read; ++tries) {
      if (tries) __builtin_amdgcn_s_sleep(2);
      read = __hip_atomic_load(flags + readers.first + tid, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != 0;
    }
  }
  if (!__syncthreads_and(read)) {   // given up: NaN in the chunk's places, of every type, and the list says so (nobody else reads its entries)
    for (int i = tid; i < count; i += 256) p.kept[(size_t)row * p.keep + first + i] = kEvictAbandoned;
#pragma unroll 1
    for (int at = line; at < count; at += 256 / LANES) {
      const u32x4 nan = {~0u, ~0u, ~0u, ~0u};
      *reinterpret_cast<u32x4*>(keys + row_at(to[at], c.key_page) + piece) = nan;
      *reinterpret_cast<u32x4*>(values + row_at(to[at], c.value_page) + piece) = nan;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int at = line + i * (256 / LANES);
    if (at >= count) break;
    const int place = to[at];
    *reinterpret_cast<u32x4*>(keys + row_at(place, c.key_page) + piece) = k[i];
    *reinterpret_cast<u32x4*>(values + row_at(place, c.value_page) + piece) = v[i];
  }
  if constexpr (E8) {
    if (tid < count) key_exponents[exponent_at(to[tid])] = ke, value_exponents[exponent_at(to[tid])] = ve;
  }
}

// Bounds of the pages that a cut row's tokens are in now, a workgroup each: a thread has a feature and tokens SIDE apart; they meet in LDS.  Bound by its loads,
// of an element a lane each (64 sequences to 2048 tokens, 8 key heads of 128: 126 us for 189 MB, 1.5 TB/s; e4m3 86).
template <bool BF16, int D, bool E8>
__global__ __launch_bounds__(256) void evict_bounds_kernel(EvictParams p) {
  constexpr int SIDE = 256 / D;
  __shared__ float low[256], high[256];
  const PagedParams& c = p.cache;
  const int rows = c.seqs * c.kv_heads, row = blockIdx.x % rows, number = blockIdx.x / rows, seq = row / c.kv_heads, head = row % c.kv_heads;
  if (p.tokens[row] == 0) return;
  const int page = c.table[(size_t)seq * c.table_row + number], count = min(1 << c.page_shift, p.keep - (number << c.page_shift));
  const int f = threadIdx.x % D;
  const size_t first = (size_t)head << c.page_shift;
  float lo = INFINITY, hi = -INFINITY;
  for (int i = threadIdx.x / D; i < count; i += SIDE) {
    float x;
    if constexpr (E8) {
      const unsigned code = static_cast<const unsigned char*>(c.keys)[page * c.key_page + (long long)(first + i) * D + f];
      const float up = power_of_two(c.key_exponents[(((size_t)page * c.kv_heads) << c.page_shift) + first + i]);
      x = f32_of_16<BF16>((unsigned short)pack_pair<BF16>(__builtin_amdgcn_cvt_f32_fp8(code, 0) * up, 0.f));
    } else {
      x = f32_of_16<BF16>(static_cast<const unsigned short*>(c.keys)[page * c.key_page + (long long)(first + i) * D + f]);
    }
    lo = smaller(lo, x), hi = larger(hi, x);
  }
  low[threadIdx.x] = lo, high[threadIdx.x] = hi;
  __syncthreads();
  if (threadIdx.x >= D) return;
#pragma unroll
  for (int i = 1; i < SIDE; ++i) lo = smaller(lo, low[f + i * D]), hi = larger(hi, high[f + i * D]);
  unsigned short* const to = p.bounds + ((size_t)page * c.kv_heads + head) * (2 * D) + f;
  to[0] = (unsigned short)pack_pair<BF16>(lo, 0.f), to[D] = (unsigned short)pack_pair<BF16>(hi, 0.f);
}

int row_bytes(const iex_paged_cache& c) { return c.head_dim * (c.eight_bits ? 1 : 2); }
int chunk_of(const iex_paged_cache& c) { return evict_chunk(row_bytes(c)); }

template <int D, bool E8>
void launch_move(const EvictParams& p, unsigned grid, hipStream_t s) {
  note_kernel("evict_move_kernel<%d, %s>", D, E8 ? "e4m3" : "16");
  hipLaunchKernelGGL((evict_move_kernel<D * (E8 ? 1 : 2), E8>), dim3(grid), dim3(256), 0, s, p);
}
template <bool E8>
void launch_move(const EvictParams& p, int head_dim, unsigned grid, hipStream_t s) {
  if (head_dim == 64) launch_move<64, E8>(p, grid, s);
  else if (head_dim == 128) launch_move<128, E8>(p, grid, s);
  else launch_move<256, E8>(p, grid, s);
}

template <bool BF16, bool E8>
void launch_bounds(const EvictParams& p, int head_dim, unsigned grid, hipStream_t s) {
  note_kernel("evict_bounds_kernel<%s, %d, %s>", BF16 ? "bf16" : "f16", head_dim, E8 ? "e4m3" : "16");
  if (head_dim == 64) hipLaunchKernelGGL((evict_bounds_kernel<BF16, 64, E8>), dim3(grid), dim3(256), 0, s, p);
  else if (head_dim == 128) hipLaunchKernelGGL((evict_bounds_kernel<BF16, 128, E8>), dim3(grid), dim3(256), 0, s, p);
  else hipLaunchKernelGGL((evict_bounds_kernel<BF16, 256, E8>), dim3(grid), dim3(256), 0, s, p);
}

// A table that holds no more than is kept: nothing ever moves.
bool never(const iex_paged_cache& c, int keep) { return (long long)c.table_width * c.page_size <= keep; }

struct Layout {
  long long rows, chunks;
  int slices;                                                              // of a row, 0: rows are in LDS
  size_t tickets, flags, before, kept_weights, histograms, found, bytes;   // where they begin, behind the rows' tokens
};
Layout layout_of(const iex_paged_cache& c, int keep) {
  Layout l;
  if (never(c, keep)) keep = 0;
  l.rows = (long long)c.seqs * c.kv_heads, l.chunks = ceil_div(keep, chunk_of(c));
  l.tickets = (size_t)l.rows * 4;
  l.flags = l.tickets + (size_t)l.rows * 4;
  l.before = l.flags + (size_t)l.rows * l.chunks * 4;
  l.kept_weights = l.before + (size_t)l.rows * (l.chunks + 1) * 4;
  const long long room = (long long)c.table_width * c.page_size;
  l.slices = room <= kEvictKept ? 0 : ceil_div(room, kEvictSlice);
  l.found = (l.kept_weights + (size_t)l.rows * keep * 4 + 15) / 16 * 16;
  l.histograms = l.found + (size_t)l.rows * l.slices * 16;
  l.bytes = l.histograms + (size_t)l.rows * l.slices * 2 * 256 * 4;
  return l;
}
// Workgroups of 512 threads where there are many more rows than CUs, which then have several at a time, or rows are short (both launches, 512 rows of 1024
// tokens 15.9 us, 2048 of 8192 88; by 1024 threads 17.5 and 99); else of 1024 (8 rows of 4096 16.9, 512 of 8192 32.5; by 512 18.4 and 34.5).
bool few_threads(long long rows, long long room) { return room <= 1024 || (room <= 12288 && rows * 10 > room); }

}  // namespace
}  // namespace iex

extern "C" size_t iex_evict_tokens_workspace_bytes(const iex_paged_cache* cache, int keep) {
  using namespace iex;
  if (check_paged_cache(cache, "evict_tokens", false) || keep < 1) return 0;
  return layout_of(*cache, keep).bytes;
}

extern "C" int iex_evict_tokens(const iex_paged_cache* cache, int* lengths, float* weights, int keep, int recent, int first, int* kept, void* workspace,
                                size_t workspace_bytes, void* stream) {
  return iex_evict_tokens_within(cache, lengths, weights, keep, recent, first, kept, iex::kEvictTries, workspace, workspace_bytes, stream);
}

extern "C" int iex_evict_tokens_within(const iex_paged_cache* cache, int* lengths, float* weights, int keep, int recent, int first, int* kept, int tries, void* workspace,
                                       size_t workspace_bytes, void* stream) {
  using namespace iex;
  trail_reset();
  if (int rc = check_paged_cache(cache, "evict_tokens", true)) return rc;
  IEX_REQUIRE(keep > 0 && first >= 0 && recent >= 0 && (long long)first + recent <= keep, IEX_ERR_BAD_ARGUMENT,
              "evict_tokens: at least one token, the first and recent ones that are always kept among them (keep=%d first=%d recent=%d)", keep, first, recent);
  IEX_REQUIRE(tries >= 0 && tries <= kEvictTries, IEX_ERR_BAD_ARGUMENT, "evict_tokens: a wait of 0 to %d looks (%d)", kEvictTries, tries);
  if (cache->seqs == 0 || cache->kv_heads == 0) return 0;
  IEX_REQUIRE(lengths == cache->lengths && kept && (weights || cache->table_width == 0), IEX_ERR_BAD_ARGUMENT, "evict_tokens: null pointer argument");
  IEX_REQUIRE(aligned(weights, 16), IEX_ERR_UNSUPPORTED, "evict_tokens: the weights must be 16-byte aligned");
  IEX_REQUIRE(aligned(kept, 4), IEX_ERR_UNSUPPORTED, "evict_tokens: operands must be aligned to their elements");
  IEX_REQUIRE((long long)cache->pages * cache->page_size < (1ll << 31), IEX_ERR_TOO_LARGE, "evict_tokens: up to 2^31 tokens in a cache");
  const Layout l = layout_of(*cache, keep);
  const bool moves = !never(*cache, keep) && cache->pages > 0;
  const long long pages = moves && cache->bounds ? ceil_div(keep, cache->page_size) : 0;   // whose bounds change
  IEX_REQUIRE(l.rows < (1ll << 22) && l.rows * l.slices < (1ll << 22) && l.rows * l.chunks < (1ll << 24) && l.rows * pages < (1ll << 24), IEX_ERR_TOO_LARGE,
              "evict_tokens: too many sequences, heads or tokens to keep");
  IEX_REQUIRE(workspace && aligned(workspace, 256) && workspace_bytes >= l.bytes, IEX_ERR_BAD_ARGUMENT, "evict_tokens: needs a 256-byte aligned workspace of %zu bytes", l.bytes);
  EvictParams p{};
  p.cache = paged_params(*cache);
  p.keep = keep, p.first = first, p.recent = recent, p.chunks = (int)l.chunks, p.tries = tries;
  p.lengths = lengths, p.weights = weights, p.kept = kept, p.bounds = static_cast<unsigned short*>(cache->bounds);
  char* const ws = static_cast<char*>(workspace);
  p.tokens = reinterpret_cast<int*>(ws), p.tickets = reinterpret_cast<int*>(ws + l.tickets), p.flags = reinterpret_cast<int*>(ws + l.flags);
  p.before = reinterpret_cast<int*>(ws + l.before), p.kept_weights = reinterpret_cast<float*>(ws + l.kept_weights);
  hipStream_t s = static_cast<hipStream_t>(stream);
  p.found = reinterpret_cast<int4*>(ws + l.found), p.histograms = reinterpret_cast<unsigned*>(ws + l.histograms), p.slices = l.slices;
  const long long room = (long long)cache->table_width * cache->page_size;
  const size_t lds = room * 4;
  const int chunk_shift = log2_of(chunk_of(*cache));   // (a power of two)
  if (l.slices) {
    note_kernel("evict_slice_kernel x 5");
    const dim3 slices((unsigned)(l.rows * l.slices)), threads(kEvictThreads);
    hipLaunchKernelGGL((evict_slice_kernel<0>), slices, threads, 0, s, p, chunk_shift);
    hipLaunchKernelGGL((evict_slice_kernel<1>), slices, threads, 0, s, p, chunk_shift);
    hipLaunchKernelGGL((evict_slice_kernel<2>), slices, threads, 0, s, p, chunk_shift);
    hipLaunchKernelGGL((evict_slice_kernel<3>), slices, threads, 0, s, p, chunk_shift);
    hipLaunchKernelGGL((evict_slice_kernel<4>), slices, threads, 0, s, p, chunk_shift);
  } else {
    note_kernel("evict_select_kernel");
    if (lds > 48 * 1024) {   // (beside what the selection has)
      static thread_local unsigned long long raised = 0;   // on which devices
      int device = 0;
      if (int rc = check_hip(hipGetDevice(&device), "hipGetDevice")) return rc;
      if (!(raised >> (device & 63) & 1)) {
        if (int rc = check_hip(hipFuncSetAttribute(reinterpret_cast<const void*>(evict_select_kernel<kEvictThreads>), hipFuncAttributeMaxDynamicSharedMemorySize, kEvictKept * 4),
                               "hipFuncSetAttribute(LDS size)"))
          return rc;
        raised |= 1ull << (device & 63);
      }
    }
    if (few_threads(l.rows, room)) hipLaunchKernelGGL((evict_select_kernel<512>), dim3((unsigned)l.rows), dim3(512), lds, s, p, chunk_shift);
    else hipLaunchKernelGGL((evict_select_kernel<kEvictThreads>), dim3((unsigned)l.rows), dim3(kEvictThreads), lds, s, p, chunk_shift);
  }
  if (int rc = check_hip(hipGetLastError(), "evict_tokens launch")) return rc;
  if (!moves) return 0;
  const unsigned grid = (unsigned)(l.rows * l.chunks);
  if (cache->eight_bits) launch_move<true>(p, cache->head_dim, grid, s);
  else launch_move<false>(p, cache->head_dim, grid, s);
  if (int rc = check_hip(hipGetLastError(), "evict_tokens launch")) return rc;
  if (!pages) return 0;
  const unsigned page_grid = (unsigned)(l.rows * pages);
  if (cache->dtype == IEX_BF16) cache->eight_bits ? launch_bounds<true, true>(p, cache->head_dim, page_grid, s) : launch_bounds<true, false>(p, cache->head_dim, page_grid, s);
  else cache->eight_bits ? launch_bounds<false, true>(p, cache->head_dim, page_grid, s) : launch_bounds<false, false>(p, cache->head_dim, page_grid, s);
  return check_hip(hipGetLastError(), "evict_tokens launch");
}
