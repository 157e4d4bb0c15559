// Attention of one new token per sequence over a paged cache: out = softmax(scale q k^T) v over the cache's tokens, per query
// head; the query heads of a group share a key head.
//
// Every key and value is read once and multiplied with at most 16 queries: memory is what bounds it, so the design keeps loads in
// flight and everything else out of their way.  Tiles of 32 or 64 tokens go from the pages straight into registers as matrix-core
// operands, no LDS:
//   S^T = K Q^T    MFMA rows = tokens, columns = queries: a lane's operand is 16 bytes of one token's key.  Lane (column c, group
//                  g = lane / 16) gets the scores of query c with tokens 4g .. 4g + 3 of each 16 ...
//   O^T += V^T P^T ... and its eight probabilities of 32 tokens are the operand of the product with the values, no lane exchange,
//                  if group g's share of the sum over tokens is those very tokens.  A lane loads 16 bytes (features c * 8 ..) of
//                  each of them; one byte permute per dword pairs tokens, and operand j has features c * 8 + j as its rows.
// The running maximum and sum are per query; sums follow a new maximum only where some score has passed it.  Probabilities go
// in as 16-bit parts, three of bf16 (all of their 24 bits) or two of fp16 (22): matrix cores idle otherwise.
//
// A sequence is split over its length into parts, a workgroup each (paged_cache.h: parts are cut from the lengths on the device,
// so a replayed graph follows them); one, four or eight wavefronts take its tiles in turn and meet in LDS, parts meet in a second launch.
// An 8-bit cache (e4m3) widens to 16 bits in registers; its powers of two go to the scores and the probabilities.
//
// Measured: 131071 tokens, 8 key heads of 128, 64 query heads, bf16 88 us = 6.2 TB/s, its join 6; 64 sequences of 4000 .. 16384 in e4m3
// 200 us = 6.0 TB/s; 16 x 600 .. 1023, 32 heads 40 us = 5.3; 16 x 1007 .. 1693, 16 heads of 256 63.5 us = 5.7; 128 x 1 .. 4096, 16 heads of 64,
// pages of 16 55 us = 4.9 (vector units busy 9 - 37 %, matrix cores 4 - 14 %; profiles/paged_cache_kernel_trace_and_counters.txt).
#pragma once
#include "paged_cache_device.cuh"

namespace iex {

struct PagedAttentionParams {
  PagedParams cache;
  int heads, group, group_tiles;   // query heads, those of a key head, blocks of 16 of them
  int pitch, count;                // query rows of a part's result; pages listed per sequence and key head, 0: all of the table
  int blocks, slots;               // blocks of up to 16 query heads of a key head; parts beyond one per sequence
  int few;                         // tiles (of all sequences) that get a workgroup each
  int fixed;                       // parts of every row, where that does not go by the lengths (whole rows, listed pages); else 0
  const int* listed;
  const unsigned short* q;
  unsigned short* out;
  long long q_strides[3], out_strides[3];   // sequence, head, feature
  bool q_rows;
  float scale_log2;
  float* partial;   // per part: group_rows x D sums, then per part group_rows maxima and sums
  float* stats;
  // attention that keeps account (WEIGH below)
  float* weights;     // (seqs, kv_heads, tokens of a table)
  float* scores;      // (seqs, kv_heads, tokens of a table / 16, heads of a key head, 16): what a wavefront leaves of a tile lies together
  float* row_stats;   // per sequence and query head maximum and sum, of rows of one part
  int at_once;        // rows are whole and their queries together: no second launch
};

__device__ __forceinline__ size_t table_tokens(const PagedParams& c) { return (size_t)c.table_width << c.page_shift; }
// The scores of a sequence and key head; query i's with four tokens from t on are at account_place(t, i).
__device__ __forceinline__ float* account_scores(const PagedAttentionParams& p, int seq, int kv_head) {
  return p.scores + ((size_t)seq * p.cache.kv_heads + kv_head) * table_tokens(p.cache) * p.group;
}
__device__ __forceinline__ size_t account_place(const PagedAttentionParams& p, int t, int i) { return (size_t)(t & ~15) * p.group + i * 16 + (t & 15); }

// What stands in the place of the score of a token that is not attended to: a NaN that no product of 16-bit or 8-bit operands has, so that a row whose
// scores are NaN or infinite leaves no trace in what it does not attend to.
constexpr unsigned kNoScore = 0xFFFFFFFFu;

// exp2((score - maximum) * scale) is taken as exp2(score * scale - maximum * scale) in one fused step, whose second product is rounded: to 2^-8 at 2^16, by
// more where it is larger, up to what leaves 16 bits, or 32 (fp16 heads of 128 of values around 10^4: infinite results).  Beyond, the difference comes first.
constexpr float kFarShift = 65536.f;

// Four tokens' scores of one query as weights: exp2((score - maximum) * scale) / sum.
struct QueryWeights {
  float top, share;
  __device__ __forceinline__ QueryWeights(float maximum, float sum) : top(sum == -1.f ? 0.f : maximum), share(sum == -1.f ? 0.f : 1.f / sum) {}
  __device__ __forceinline__ QueryWeights(float2 both) : top(both.x), share(both.y) {}
  __device__ __forceinline__ void add(f32x4& to, const f32x4& score, float scale_log2) const {
    const float product = -top * scale_log2;
    const bool far = fabsf(product) > kFarShift;
    const float first = far ? top : 0.f, shift = far ? 0.f : product;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float more = fmaf(__builtin_amdgcn_exp2f(fmaf(score[r] - first, scale_log2, shift)), share, to[r]);
      to[r] = __float_as_uint(score[r]) == kNoScore ? to[r] : more;
    }
  }
};
// `got` more for tokens t .. t + 3 of a row of `length` (the others are not touched).
__device__ __forceinline__ void add_weights(float* weights, int t, int length, const f32x4& got) {
  if (t + 4 <= length) {
    f32x4 now = *reinterpret_cast<f32x4*>(weights + t);
#pragma unroll
    for (int r = 0; r < 4; ++r) now[r] += got[r];
    *reinterpret_cast<f32x4*>(weights + t) = now;
  } else {
    for (int r = 0; t + r < length; ++r) weights[t + r] += got[r];
  }
}

// Tokens that a sequence of `length` tokens attends to at most.
__device__ __forceinline__ int row_tokens(const PagedAttentionParams& p, int length) { return p.count && length ? p.count << p.cache.page_shift : length; }

// What weights, 1 at most, are multiplied with on their way to the values, and the sum of them when it divides.  Before bf16 and e4m3 values
// they come to 1 at most all together, so that their sums stay within the values' range (two values of 2e38 came out infinite); before
// fp16 values, far from 32 bits' ends, they go up to 2^15, so that small ones are not below fp16's range.
__device__ __forceinline__ float weight_scale(bool range_of_bf16, int tokens) {
  return power_of_two(range_of_bf16 ? 127 - (tokens > 1 ? 32 - __builtin_clz(tokens - 1) : 0) : 127 + 15);
}

// The lengths of 64 sequences, one a lane.
struct LaneLengths {
  int from = -kWave, mine = 0;
  __device__ __forceinline__ void load(const PagedParams& c, int first) {
    const int s = first + lane_id();
    from = first;
    mine = s < c.seqs ? cached_length(c.lengths[s], c.table_width, 1 << c.page_shift) : 0;
  }
  __device__ __forceinline__ int of(const PagedParams& c, int seq) {
    if (seq < from || seq >= from + kWave) load(c, seq);
    return bcast_i(mine, seq - from);
  }
};
__device__ __forceinline__ int lane_tiles(const PagedAttentionParams& p, const LaneLengths& l) { return l.from + lane_id() < p.cache.seqs ? paged_tiles(l.mine) : 0; }

// The first sequence that `match` says yes to (its number, its first part's, its parts), by the lengths; `lengths` holds its.
template <typename MATCH>
__device__ __forceinline__ bool find_part(const PagedAttentionParams& p, LaneLengths& lengths, MATCH match, int& seq, int& first, int& parts, int& tiles) {
  int total = 0;
  for (int s0 = 0; s0 < p.cache.seqs; s0 += kWave) {
    lengths.load(p.cache, s0);
    total += lane_tiles(p, lengths);
  }
  total = bcast_i(wave_scan(total), kWave - 1);
  const int most = paged_part_most(total - p.cache.seqs, p.slots, paged_least(total, p.few));
  int before = 0;
  for (int s0 = 0; s0 < p.cache.seqs; s0 += kWave) {
    if (p.cache.seqs > kWave) lengths.load(p.cache, s0);
    const int mine = lane_tiles(p, lengths), n = s0 + lane_id() < p.cache.seqs ? paged_parts(mine, most) : 0, upto = before + wave_scan(n);
    const unsigned long long hit = __ballot(match(s0 + lane_id(), upto - n, n));
    if (hit) {
      const int lane = __ffsll(hit) - 1;
      seq = s0 + lane, first = bcast_i(upto - n, lane), parts = bcast_i(n, lane), tiles = bcast_i(mine, lane);
      return true;
    }
    before = bcast_i(upto, kWave - 1);
  }
  return false;
}

// Two e4m3 codes of a dword to a pair of 16-bit values (exact).
template <bool BF16, bool HIGH>
__device__ __forceinline__ unsigned widen_pair(unsigned codes) {
  if constexpr (BF16) return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, 1.f, HIGH));
  else return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, 1.f, HIGH));
}

// Two weights as 16-bit parts whose sum they are: three of bf16 hold all 24 bits, two of fp16 22 (a difference of 2^-22 beside a result
// rounded at 2^-11).  Two of bf16 would hold 16, and results then differ more often by a bit from what 32-bit weights give (1.1e-4 of them in
// place of 1.9e-5 over 64 pages of 64 tokens; the third part is 61.4 -> 61.9 us of 128 x 1 .. 4096 tokens in heads of 64, 206.4 -> 208.2 of
// 64 x 4000 .. 16384 in e4m3).  Where values can be infinite (16-bit caches) every part is positive: all but the last are rounded down and none
// is zero (the weight's lowest bit is set, and a last part that would be zero is the smallest there is), so that weight times infinity is
// infinity and not inf - inf or 0 inf (in fp16 down to 2^-16 of the row's largest weight, in bf16 2^-80: below, a part can be lost).
template <bool BF16>
constexpr int kWeightParts = BF16 ? 3 : 2;
template <bool BF16, bool E8>
__device__ __forceinline__ void split_pair(float a, float b, unsigned (&part)[kWeightParts<BF16>]) {
  constexpr int N = kWeightParts<BF16>;
  if constexpr (!E8) a = __uint_as_float(__float_as_uint(a) | 1u), b = __uint_as_float(__float_as_uint(b) | 1u);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (E8 || i == N - 1) part[i] = pack_pair<BF16>(a, b);
    else if constexpr (BF16) part[i] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
    else part[i] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_pkrtz(a, b));
    if (i == N - 1) break;
    float a0, b0;
    unpack_pair<BF16>(part[i], a0, b0);
    a -= a0, b -= b0;
    if (!E8 && i == 1) a = fmaxf(a, 0x1p-126f), b = fmaxf(b, 0x1p-126f);   // (the first rest has the lowest bit)
  }
}

// A load, with the streaming hint where what is read is far larger than the caches.
template <bool STREAM, typename T>
__device__ __forceinline__ T load_from(const T* p) {
  if constexpr (STREAM) return __builtin_nontemporal_load(p);
  else return *p;
}

// Places of 16 tokens of a wavefront's tile.  (Heads of 64 in 16 bits by four: 512 x 16 rows of 128 tokens 54.5 -> 63.7 us.)
constexpr int paged_places(int head_dim, bool eight_bits) { return eight_bits && head_dim <= 128 ? 4 : 2; }
// Wavefronts of a SIMD that the registers are cut for.
constexpr int paged_simd_waves(int head_dim) { return head_dim == 256 ? 2 : head_dim == 128 ? 3 : 4; }

// Rows of the wavefronts' sums in LDS: quarters 16 words further apart and an odd pitch, so that the 64 lanes, which have four features of
// 16 queries, write to 64 banks (unpadded, up to all of them to one: two sequences of 224 tokens, 16 heads of 256 17.6 us, so 15.0).
constexpr int paged_sum_gap(int head_dim) { return head_dim == 64 ? 0 : 16; }
constexpr int paged_sum_pitch(int head_dim) { return head_dim + 3 * paged_sum_gap(head_dim) + 1; }

// WEIGH: scores are left behind too, 4 bytes a token and query head, and become weights when the row's maximum and sum are known: here, by the
// one workgroup that has the row, or in paged_account_kernel.  (64 x 2049 .. 4224 tokens, 32 heads over 8: 166 us, 132 without these 25 MB of
// stores; a row for every head instead of tiles 168, held back in LDS to the end of a part 162, and then 700 tokens 13.2 for 12.4, by buffer address without a
// branch 168, past the caches 171.)
template <bool BF16, int D, bool E8, int WAVES, bool WEIGH>
__global__ __launch_bounds__(WAVES * 64, paged_simd_waves(D)) void paged_attention_kernel(PagedAttentionParams p) {
  typedef unsigned short u16;
  constexpr int ES = E8 ? 1 : 2;               // bytes of an element
  constexpr int KS = D / 32;                   // steps of the sum over features
  constexpr int KW = D * ES / 64;              // 16-byte loads of a lane for the keys of 16 tokens (E8: each is two steps)
  constexpr int F = D / 16;                    // features of a value row that a lane has: operands of the second product
  constexpr int VD = F * ES / 4, VWORDS = VD == 8 ? 2 : 1;   // ... in dwords: 1, 2, 4 or 8
  typedef std::conditional_t<VD == 1, unsigned, std::conditional_t<VD == 2, u32x2, u32x4>> VWord;
  constexpr int SUB = paged_places(D, E8);     // places of 16 tokens of a tile
  // Queries stay in LDS (a column without one has the last one's, its results are not used): with them in registers a SIMD has room for
  // one wavefront only (256 rows of 1007 .. 1693 tokens, 16 heads 123 -> 102 us; 64 of 8192 86 -> 88).
  constexpr bool Q_LDS = D == 256 && !E8;
  constexpr bool PV_BF16 = BF16 || E8;         // (an e4m3 value's power of two goes to the probability, which fp16 has not the range for)
  extern __shared__ __align__(16) float smem[];
  const int wave = uniform(threadIdx.x >> 6);
  const PagedParams& cache = p.cache;
  LaneLengths lengths;

  // ---- whose part ----
  const int block = blockIdx.x % p.blocks, item = blockIdx.x / p.blocks;
  int seq = item, part = 0, parts = 1, tiles = 1;
  const int lane = threadIdx.x & 63, entries = p.count ? p.count : cache.table_width;
  const int kv_head = block / p.group_tiles, group_tile = block % p.group_tiles;
  auto entry_at = [&](int e) -> int {   // of the sequence's list, or of its table
    if (e >= entries) return -1;
    return p.count ? p.listed[((size_t)seq * cache.kv_heads + kv_head) * p.count + e] : cache.table[(size_t)seq * cache.table_row + e];
  };
  int first_entry = 0, first_found = -1;
  if (p.fixed) {
    parts = p.fixed, seq = item / parts, part = item % parts;
    if (p.count) {
      tiles = paged_tiles(p.count << cache.page_shift);
      first_entry = paged_place(paged_part_begin(tiles, parts, part) * kPagedTile, cache.page_shift).entry;
    }
    first_found = entry_at(first_entry + lane);   // (beside the lengths, which it does not need)
    lengths.load(cache, seq);
    if (!p.count) tiles = paged_tiles(lengths.of(cache, seq));
  } else if (!find_part(p, lengths, [&](int, int first, int n) { return first + n > item; }, seq, part, parts, tiles)) {
    return;
  } else {
    part = item - part;
  }
  const int col = lane & 15, g = lane >> 4;
  const int rows = min(16, p.group - group_tile * 16);   // queries
  const int length = lengths.of(cache, seq), tokens = row_tokens(p, length);
  const float up = weight_scale(PV_BF16, tokens);
  const int begin = paged_part_begin(tiles, parts, part) * kPagedTile;
  int end = min(tokens, paged_part_begin(tiles, parts, part + 1) * kPagedTile);

  // ---- queries: columns of the first product ----
  // Rows of aligned chunks go straight into registers, queries of other strides through LDS.
  u32x4 fq[Q_LDS ? 1 : KS];
  auto feature = [&](int s) { return E8 ? s / 2 * 64 + g * 16 + s % 2 * 8 : s * 32 + g * 8; };
  u16* const q_rows = reinterpret_cast<u16*>(smem);   // (D + 8 apart: 16 columns are in different banks)
  if (Q_LDS || !p.q_rows) {
    for (int i = threadIdx.x; i < rows * (D / 8); i += WAVES * 64) {
      const int row = i / (D / 8), d = i % (D / 8) * 8;
      const u16* q = p.q + seq * p.q_strides[0] + (long long)(kv_head * p.group + group_tile * 16 + row) * p.q_strides[1];
      u32x4 x;
      if (p.q_rows) {
        x = *reinterpret_cast<const u32x4*>(q + d);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = q[(d + 2 * j) * p.q_strides[2]] | (unsigned)q[(d + 2 * j + 1) * p.q_strides[2]] << 16;
      }
      *reinterpret_cast<u32x4*>(q_rows + row * (D + 8) + d) = x;
    }
    __syncthreads();
  }
  if constexpr (!Q_LDS) {
#pragma unroll
    for (int s = 0; s < KS; ++s) fq[s] = u32x4{0u, 0u, 0u, 0u};
    if (!p.q_rows) {
      if (col < rows) {
#pragma unroll
        for (int s = 0; s < KS; ++s) fq[s] = *reinterpret_cast<const u32x4*>(q_rows + col * (D + 8) + feature(s));
      }
      __syncthreads();   // (the wavefronts' results go there)
    } else if (col < rows) {
      const u16* q = p.q + seq * p.q_strides[0] + (long long)(kv_head * p.group + group_tile * 16 + col) * p.q_strides[1];
#pragma unroll
      for (int s = 0; s < KS; ++s) fq[s] = *reinterpret_cast<const u32x4*>(q + feature(s));
    }
  }

  // ---- the pages of the part: 64 entries of the table (or list) in the lanes ----
  int window = -(1 << 30), entry_logical = 0, entry_page = -1;
  auto take_entries = [&](int from, int found) {
    window = from, entry_logical = from + lane, entry_page = found;
    if (p.count) {
      entry_logical = found, entry_page = -1;
      if ((unsigned)found < (unsigned)cache.table_width) entry_page = cache.table[(size_t)seq * cache.table_row + found];
      else entry_logical = 0;
    }
  };
  if (p.fixed) take_entries(first_entry, first_found);
  if (p.count && paged_place(end - 1, cache.page_shift).entry < window + kWave) {   // nothing behind the last page that is there (a sequence of fewer pages)
    const unsigned long long there = __ballot((unsigned)entry_page < (unsigned)cache.pages);
    end = min(end, (window + (there ? 64 - __builtin_clzll(there) : 0)) << cache.page_shift);
  }

  // Where a tile's tokens lie, 16 at a place.  Loads take no branch: what is not attended to is read from a place that exists and
  // masked where it is used.
  struct Where {
    int page[SUB], row[SUB], valid[SUB];
  };
  auto find = [&](int t) {
    Where w;
#pragma unroll
    for (int a = 0; a < SUB; ++a) {
      const PagedPlace place = paged_place(t + a * 16, cache.page_shift);
      if (place.entry >= window + kWave) take_entries(place.entry, entry_at(place.entry + lane));
      const int page = bcast_i(entry_page, place.entry - window), logical = bcast_i(entry_logical, place.entry - window);
      w.valid[a] = place.entry < entries ? paged_valid(logical, place.slot, cache.page_shift, page, cache.pages, length) : 0;
      w.page[a] = page, w.row[a] = (kv_head << cache.page_shift) + place.slot;
      if (w.valid[a] == 0) w.page[a] = a ? w.page[a ? a - 1 : 0] : 0, w.row[a] = a ? w.row[a ? a - 1 : 0] : w.row[a];
    }
    return w;
  };
  u32x4 key[SUB][KW];
  VWord value[SUB][4][VWORDS];
  typedef unsigned Places __attribute__((ext_vector_type(SUB)));
  Places ke, ve;   // exponents of this lane's four tokens at each place
  auto load_keys = [&](const Where& w) {
#pragma unroll
    for (int a = 0; a < SUB; ++a) {
      const unsigned char* k = static_cast<const unsigned char*>(cache.keys) + (w.page[a] * cache.key_page + (long long)w.row[a] * D) * ES;
#pragma unroll
      for (int s = 0; s < KW; ++s) key[a][s] = load_from<WAVES == 4>(reinterpret_cast<const u32x4*>(k + (col * (D * ES) + s * 64 + g * 16)));
      if constexpr (E8)
        ke[a] = *reinterpret_cast<const unsigned*>(cache.key_exponents + (((long long)w.page[a] * cache.kv_heads) << cache.page_shift) + w.row[a] + g * 4);
    }
  };
  auto load_values = [&](const Where& w) {
#pragma unroll
    for (int a = 0; a < SUB; ++a) {
      const unsigned char* v = static_cast<const unsigned char*>(cache.values) + (w.page[a] * cache.value_page + (long long)w.row[a] * D) * ES;
      // (heads of 256 in 16 bits: two halves of 128, so that a load of 16 lanes is 256 consecutive bytes)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int h = 0; h < VWORDS; ++h) value[a][i][h] = load_from<WAVES == 4>(reinterpret_cast<const VWord*>(v + ((g * 4 + i) * (D * ES) + h * 256 + col * (int)sizeof(VWord))));
      if constexpr (E8)
        ve[a] = *reinterpret_cast<const unsigned*>(cache.value_exponents + (((long long)w.page[a] * cache.kv_heads) << cache.page_shift) + w.row[a] + g * 4);
    }
  };
  auto value_dword = [&](int a, int r, int d) -> unsigned {
    if constexpr (VD == 1) return value[a][r][0];
    else return value[a][r][d / 4][d % 4];
  };

  f32x4 o[F];
#pragma unroll
  for (int j = 0; j < F; ++j) o[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  float top = -INFINITY, sum = 0.f;   // of this lane's query: the maximum so far (all groups'), this group's share of the sum
  int attended = 0;

  f32x4 s[SUB];
  auto scores = [&]() {
#pragma unroll
    for (int a = 0; a < SUB; ++a) s[a] = f32x4{0.f, 0.f, 0.f, 0.f};
    int q_at = (min(col, rows - 1) * (D + 8) + g * 8) * 2;
    if constexpr (Q_LDS) asm volatile("" : "+v"(q_at));   // (else all of them would be read ahead of the loop, into registers)
#pragma unroll
    for (int e = 0; e < KS; ++e) {
      u32x4 f;
      if constexpr (Q_LDS) f = *reinterpret_cast<const u32x4*>(reinterpret_cast<const unsigned char*>(smem) + q_at + e * 64);
      else f = fq[e];
#pragma unroll
      for (int a = 0; a < SUB; ++a) {
        u32x4 fk;
        if constexpr (E8) {
          const unsigned c0 = key[a][e / 2][e % 2 * 2], c1 = key[a][e / 2][e % 2 * 2 + 1];
          fk = u32x4{widen_pair<BF16, false>(c0), widen_pair<BF16, true>(c0), widen_pair<BF16, false>(c1), widen_pair<BF16, true>(c1)};
        } else {
          fk = key[a][e];
        }
        s[a] = mfma_16x16x32<BF16>(fk, f, s[a]);
      }
    }
    if constexpr (E8) {
#pragma unroll
      for (int a = 0; a < SUB; ++a)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[a][r] *= power_of_two(ke[a] >> (r * 8) & 0xFFu);
    }
  };
  constexpr int PARTS = kWeightParts<PV_BF16>;
  u32x4 weight[SUB / 2][PARTS];
  auto weights = [&](const Where& w, int t) {
    int valid = 0;
#pragma unroll
    for (int a = 0; a < SUB; ++a) valid += w.valid[a];
    attended += valid;
    if (valid != SUB * 16) {   // (uniform) tokens that are not attended to leave no trace, infinities and NaN included
#pragma unroll
      for (int a = 0; a < SUB; ++a)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (g * 4 + r >= w.valid[a]) {
            s[a][r] = -INFINITY;
#pragma unroll
            for (int h = 0; h < VWORDS; ++h) value[a][r][h] = VWord{};
            if constexpr (E8) ve[a] = (ve[a] & ~(0xFFu << (r * 8))) | 0x7Fu << (r * 8);
          }
    }
    if constexpr (WEIGH) {
      if (col < rows) {
        // (the tile's place in scalar registers, the lane's within it)
        unsigned char* const to = reinterpret_cast<unsigned char*>(account_scores(p, seq, kv_head) + (long long)t * p.group);
        const unsigned in_tile = ((group_tile * 16 + col) * 16 + g * 4) * 4;
#pragma unroll
        for (int a = 0; a < SUB; ++a)
          if (t + a * 16 < end) {
            f32x4 left = s[a];
            if (w.valid[a] != 16) {
#pragma unroll
              for (int r = 0; r < 4; ++r) left[r] = g * 4 + r >= w.valid[a] ? __uint_as_float(kNoScore) : left[r];
            }
            *reinterpret_cast<f32x4*>(to + (size_t)a * 64 * p.group + in_tile) = left;
          }
      }
    }
    float m = s[0][0];
#pragma unroll
    for (int a = 0; a < SUB; ++a)
#pragma unroll
      for (int r = 0; r < 4; ++r) m = fmaxf(m, s[a][r]);
    if (__ballot(m > top)) {
      m = fmaxf(m, __shfl_xor(m, 16));
      m = fmaxf(m, __shfl_xor(m, 32));
      if (m > top) {
        const float keep = __builtin_amdgcn_exp2f((top - m) * p.scale_log2);
        top = m;
        sum *= keep;
#pragma unroll
        for (int j = 0; j < F; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) o[j][r] *= keep;
      }
    }
    float shift = top == -INFINITY ? 0.f : -top * p.scale_log2;
    if (__ballot(fabsf(shift) > kFarShift)) {   // (of some query)
      const bool far = fabsf(shift) > kFarShift;
#pragma unroll
      for (int a = 0; a < SUB; ++a)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[a][r] -= far ? top : 0.f;
      shift = far ? 0.f : shift;
    }
#pragma unroll
    for (int a = 0; a < SUB; ++a) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[a][r] = __builtin_amdgcn_exp2f(fmaf(s[a][r], p.scale_log2, shift));   // (exp2(-infinity) = 0)
        sum += s[a][r];
        s[a][r] *= E8 ? power_of_two(ve[a] >> (r * 8) & 0xFFu) * up : up;
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        unsigned part[PARTS];
        split_pair<PV_BF16, E8>(s[a][2 * r], s[a][2 * r + 1], part);
#pragma unroll
        for (int i = 0; i < PARTS; ++i) weight[a / 2][i][a % 2 * 2 + r] = part[i];
      }
    }
  };
  auto weigh_values = [&]() {
#pragma unroll
    for (int j = 0; j < F; ++j)
#pragma unroll
      for (int two = 0; two < SUB / 2; ++two) {
        u32x4 fv;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int a = two * 2 + w / 2, r = w % 2 * 2;   // tokens r and r + 1 of the four at place a
          if constexpr (E8) {
            // byte j of both rows side by side, then widened
            const unsigned pair = __builtin_amdgcn_perm(value_dword(a, r + 1, j / 4), value_dword(a, r, j / 4), (j % 4) | (4 + j % 4) << 8);
            fv[w] = widen_pair<PV_BF16, false>(pair);
          } else {
            fv[w] = __builtin_amdgcn_perm(value_dword(a, r + 1, j / 2), value_dword(a, r, j / 2), j % 2 ? 0x07060302u : 0x05040100u);
          }
        }
#pragma unroll
        for (int i = 0; i < PARTS; ++i) o[j] = mfma_16x16x32<PV_BF16>(fv, weight[two][i], o[j]);
      }
  };

  // ---- the part's tiles, a wavefront's in turn.  A tile's values are asked for before its keys are waited for, the next tile's
  // keys as soon as this one's have been multiplied: half a tile is in flight at any time, in one set of registers.  (The last
  // tile is written out behind the loop, so that a wait knows on every path how many loads are behind the ones it is for.)
  int t = begin + wave * (SUB * 16);
  constexpr int STEP = WAVES * SUB * 16;
  if (t < end && cache.pages > 0) {
    Where now = find(t);
    load_keys(now);
    for (; t + STEP < end; t += STEP) {
      load_values(now);
      const Where next = find(t + STEP);
      scores();
      load_keys(next);
      weights(now, t);
      weigh_values();
      now = next;
    }
    load_values(now);
    scores();
    weights(now, t);
    weigh_values();
  }

  // ---- the wavefronts meet ----
  if constexpr (Q_LDS) __syncthreads();   // (in place of the queries)
  sum += __shfl_xor(sum, 16);
  sum += __shfl_xor(sum, 32);
  if (attended == 0) sum = -1.f;   // no token at all: zeros, whatever the formula says of an empty sum
  constexpr int PITCH = paged_sum_pitch(D), GAP = paged_sum_gap(D);
  float* sums = smem;                              // [wave][row][PITCH]
  float* tops = smem + WAVES * rows * PITCH;       // [wave][row] (maximum, sum)
  float2* shares = reinterpret_cast<float2*>(smem + (WAVES * rows * (PITCH + 2) + 1) / 2 * 2);   // WEIGH: [row]
  if (col < rows) {
    float* mine = sums + (wave * rows + col) * PITCH + g * (D / 4 + GAP);
#pragma unroll
    for (int j = 0; j < F; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        // (lane column g * 4 + r's features)
        mine[VD == 8 ? j / 8 * 32 + r * 8 + j % 8 : r * F + j] = o[j][r];
      }
    if (g == 0) tops[(wave * rows + col) * 2] = top, tops[(wave * rows + col) * 2 + 1] = sum;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < rows * D; i += WAVES * 64) {
    const int row = i / D, d = i % D, at = VD == 8 ? d % 128 / 32 * (D / 4 + GAP) + d / 128 * 32 + d % 32 : d / (D / 4) * (D / 4 + GAP) + d % (D / 4);
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) m = fmaxf(m, tops[(w * rows + row) * 2]);
    float all = 0.f, acc = 0.f;
    bool any = false;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float mine = tops[(w * rows + row) * 2], share = tops[(w * rows + row) * 2 + 1];
      if (share == -1.f) continue;
      any = true;
      const float keep = mine == m ? 1.f : __builtin_amdgcn_exp2f((mine - m) * p.scale_log2);
      all += keep * share;
      acc += keep * sums[(w * rows + row) * PITCH + at];
    }
    if (parts == 1) {
      const int head = kv_head * p.group + group_tile * 16 + row;
      p.out[seq * p.out_strides[0] + head * p.out_strides[1] + d * p.out_strides[2]] = f32_to_16(any ? acc / (all * up) : 0.f, BF16);
      if (WEIGH && d == 0 && !p.at_once) *reinterpret_cast<float2*>(p.row_stats + ((size_t)seq * p.heads + head) * 2) = float2{m, any ? all : -1.f};
      if (WEIGH && d == 0 && p.at_once) {
        const QueryWeights mine(m, any ? all : -1.f);
        shares[row] = float2{mine.top, mine.share};
      }
    } else {
      const size_t to = (size_t)blockIdx.x * p.pitch + row;
      p.partial[to * D + d] = acc;
      if (d == 0) p.stats[to * 2] = m, p.stats[to * 2 + 1] = any ? all : -1.f;
    }
  }
  if constexpr (WEIGH) {
    if (!p.at_once) return;
    __syncthreads();   // (the wavefronts' scores are there too)
    const float* from = account_scores(p, seq, kv_head);
    float* to = p.weights + ((size_t)seq * cache.kv_heads + kv_head) * table_tokens(cache);
    for (int t = threadIdx.x * 4; t < length; t += WAVES * 256) {
      f32x4 got = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
      for (int row = 0; row < rows; ++row) QueryWeights(shares[row]).add(got, *reinterpret_cast<const f32x4*>(from + account_place(p, t, row)), p.scale_log2);
      add_weights(to, t, length, got);
    }
  }
}

// Parts of a row into its result, a workgroup per sequence and query head: the parts' weights first, 256 at a time, then
// 256 / (D / 4) parts side by side, a thread four features; they meet in LDS.
template <bool BF16, int D, bool E8>
__device__ __forceinline__ void join_parts(const PagedAttentionParams& p, int seq, int head) {
  constexpr int LANES = D / 4, SIDE = 256 / LANES;   // threads of a row; parts side by side
  __shared__ float4 accs[SIDE][LANES];
  __shared__ float weights[256], tops[4], sums[4];
  const int tid = threadIdx.x;
  const int kv_head = head / p.group, in_group = head % p.group;
  LaneLengths lengths;
  int found, first = seq * p.fixed, number = p.fixed, tiles;
  if (!p.fixed && (!find_part(p, lengths, [&](int s, int, int) { return s == seq; }, found, first, number, tiles) || number == 1)) return;
  const float up = weight_scale(BF16 || E8, row_tokens(p, lengths.of(p.cache, seq)));
  const int block = kv_head * p.group_tiles + in_group / 16;
  auto place = [&](int i) { return ((size_t)(first + i) * p.blocks + block) * p.pitch + in_group % 16; };
  const int lane = tid % LANES, side = tid / LANES;
  float4 acc = {0.f, 0.f, 0.f, 0.f};
  float top = -INFINITY, total = 0.f;
  bool any = false;
  constexpr int AHEAD = 4;
  for (int i0 = 0; i0 < number; i0 += 256) {
    const int i = i0 + tid, n = min(256, number - i0);
    float4 ahead[AHEAD];   // the first parts' sums, beside the weights
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (side + k * SIDE < n) ahead[k] = *reinterpret_cast<const float4*>(p.partial + place(i0 + side + k * SIDE) * D + lane * 4);
    float m = -INFINITY, part = -1.f;
    if (i < number) {
      const float2 both = *reinterpret_cast<const float2*>(p.stats + place(i) * 2);
      m = both.x, part = both.y;
    }
    const bool counts = part != -1.f;   // (NaN is a sum)
    const float most = wave_max(counts ? m : -INFINITY);
    if (lane_id() == 0) tops[tid >> 6] = most;
    any |= __syncthreads_or(counts);
    const float now = fmaxf(fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])), top);
    const float keep = top == now ? 1.f : __builtin_amdgcn_exp2f((top - now) * p.scale_log2);
    const float weight = !counts ? 0.f : m == now ? 1.f : __builtin_amdgcn_exp2f((m - now) * p.scale_log2);
    weights[tid] = weight;
    const float share = wave_sum(counts ? weight * part : 0.f);
    if (lane_id() == 0) sums[tid >> 6] = share;
    __syncthreads();
    total = total * keep + (sums[0] + sums[1] + sums[2] + sums[3]);
    acc.x *= keep, acc.y *= keep, acc.z *= keep, acc.w *= keep;
    top = now;
    // (a part without a token left zeros)
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (side + k * SIDE < n) {
        const float w = weights[side + k * SIDE];
        acc.x = fmaf(w, ahead[k].x, acc.x), acc.y = fmaf(w, ahead[k].y, acc.y), acc.z = fmaf(w, ahead[k].z, acc.z), acc.w = fmaf(w, ahead[k].w, acc.w);
      }
#pragma unroll 4
    for (int j = side + AHEAD * SIDE; j < n; j += SIDE) {
      const float w = weights[j];
      const float4 x = *reinterpret_cast<const float4*>(p.partial + place(i0 + j) * D + lane * 4);
      acc.x = fmaf(w, x.x, acc.x), acc.y = fmaf(w, x.y, acc.y), acc.z = fmaf(w, x.z, acc.z), acc.w = fmaf(w, x.w, acc.w);
    }
    __syncthreads();
  }
  accs[side][lane] = acc;
  __syncthreads();
  if (tid >= D) return;
  float x = 0.f;
#pragma unroll
  for (int i = 0; i < SIDE; ++i) x += reinterpret_cast<const float*>(accs[i])[tid];
  p.out[seq * p.out_strides[0] + head * p.out_strides[1] + tid * p.out_strides[2]] = f32_to_16(any ? x / (total * up) : 0.f, BF16);
}
template <bool BF16, int D, bool E8>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttentionParams p) {
  join_parts<BF16, D, E8>(p, blockIdx.x, blockIdx.y);
}

// The second launch of attention that keeps account: the first workgroups add the weights of 1024 tokens at a time of a sequence and key head, `side` of
// them taking turns; the last `joins` join parts (of rows that were cut: in one launch with the weights, since neither waits for the other; each works out the
// rows' maxima and sums from the parts').  64 x 2049 .. 4224 tokens, 32 heads over 8 15.2 us (with the joins first 17.4, when this order took 14.9).
constexpr int kAccountTokens = 1024;
template <bool BF16, int D, bool E8>
__global__ __launch_bounds__(256) void paged_account_kernel(PagedAttentionParams p, int joins, int side) {
  extern __shared__ __align__(16) float2 shares[];   // of the group's queries
  const int adding = gridDim.x - joins;
  if ((int)blockIdx.x >= adding) {
    const int join = blockIdx.x - adding;
    join_parts<BF16, D, E8>(p, join / p.heads, join % p.heads);
    return;
  }
  const PagedParams& cache = p.cache;
  const int item = blockIdx.x, row = item / side, seq = row / cache.kv_heads, kv_head = row % cache.kv_heads, wave = uniform(threadIdx.x >> 6), lane = lane_id();
  const int length = cached_length(cache.lengths[seq], cache.table_width, 1 << cache.page_shift);
  int t = item % side * kAccountTokens + threadIdx.x * 4;
  if (item % side * kAccountTokens >= length) return;
  LaneLengths lengths;
  int found, first = seq, number = 1, tiles;
  if (!p.fixed) find_part(p, lengths, [&](int s, int, int) { return s == seq; }, found, first, number, tiles);
  for (int i = wave; i < p.group; i += 4) {
    const int head = kv_head * p.group + i;
    float top = -INFINITY, sum = -1.f;
    if (number == 1) {
      const float2 both = *reinterpret_cast<const float2*>(p.row_stats + ((size_t)seq * p.heads + head) * 2);
      top = both.x, sum = both.y;
    } else {
      const int block = kv_head * p.group_tiles + i / 16;
      auto part = [&](int n) { return *reinterpret_cast<const float2*>(p.stats + (((size_t)(first + n) * p.blocks + block) * p.pitch + i % 16) * 2); };
      bool counts = false;
      for (int n = lane; n < number; n += kWave)
        if (const float2 both = part(n); both.y != -1.f) counts = true, top = fmaxf(top, both.x);   // (NaN is a sum)
      top = wave_max(top);
      float mine = 0.f;
      for (int n = lane; n < number; n += kWave)
        if (const float2 both = part(n); both.y != -1.f) mine += both.x == top ? both.y : __builtin_amdgcn_exp2f((both.x - top) * p.scale_log2) * both.y;
      sum = wave_sum(mine);
      if (!__ballot(counts)) sum = -1.f;
    }
    const QueryWeights its(top, sum);
    if (lane == 0) shares[i] = float2{its.top, its.share};
  }
  __syncthreads();
  const float* from = account_scores(p, seq, kv_head);
  float* to = p.weights + ((size_t)seq * cache.kv_heads + kv_head) * table_tokens(cache);
  for (; t < length; t += side * kAccountTokens) {
    f32x4 got = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int i = 0; i < p.group; ++i) QueryWeights(shares[i]).add(got, *reinterpret_cast<const f32x4*>(from + account_place(p, t, i)), p.scale_log2);
    add_weights(to, t, length, got);
  }
}

}  // namespace iex
