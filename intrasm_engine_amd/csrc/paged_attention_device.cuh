// Attention of one new token per sequence over a paged cache: out = softmax(scale q k^T) v over the cache's tokens, per query
// head; the query heads of a group share a key head.
//
// Every key and value is read once and multiplied with at most 16 queries: memory is what bounds it, so the design keeps loads in
// flight and everything else out of their way.  Tiles of 32 tokens go from the pages straight into registers as matrix-core
// operands, no LDS:
//   S^T = K Q^T    MFMA rows = tokens, columns = queries: a lane's operand is 16 bytes of one token's key.  Lane (column c, group
//                  g = lane / 16) gets the scores of query c with tokens 4g .. 4g + 3 of each 16 ...
//   O^T += V^T P^T ... and its eight probabilities of 32 tokens are the operand of the product with the values, no lane exchange,
//                  if group g's share of the sum over tokens is those very tokens.  A lane loads 16 bytes (features c * 8 ..) of
//                  each of them; one byte permute per dword pairs tokens, and operand j has features c * 8 + j as its rows.
// The running maximum and sum are per query; sums follow a new maximum only where some score has passed it.  Probabilities go
// in as two 16-bit parts, p = hi + lo (bf16), so that they keep 16 bits: matrix cores idle otherwise, and one part rounded costs
// about half again the error of the rounded result.
//
// A sequence is split over its length into parts, a workgroup each (paged_cache.h: parts are cut from the lengths on the device,
// so a replayed graph follows them); four wavefronts take a part's tiles in turn and meet in LDS, parts meet in a second launch.
// An 8-bit cache (e4m3) widens to 16 bits in registers; its powers of two go to the scores and the probabilities.
#pragma once
#include "paged_cache_device.cuh"

namespace iex {

struct PagedAttentionParams {
  PagedParams cache;
  int heads, group, group_tiles;   // query heads, those of a key head, blocks of 16 of them
  int pitch, slots, count;         // query rows of a part's result; parts beyond one per sequence (paged_slots); pages listed per sequence and key head, 0: all of the table
  const int* listed;
  const unsigned short* q;
  unsigned short* out;
  long long q_strides[3], out_strides[3];   // sequence, head, feature
  float scale_log2;
  float* partial;   // per part: group_rows x D sums, then per part group_rows maxima and sums
  float* stats;
};

constexpr int kPagedWaves = 4, kPagedLeast = 2;   // wavefronts of a workgroup; tiles of kPagedTile tokens that are worth a part

// The sequence and part of a workgroup, from the lengths (every wavefront for itself).
struct PagedItem {
  int seq, part, parts, part_tiles, first_item;
};
__device__ __forceinline__ int paged_tokens(const PagedAttentionParams& p, int seq) {
  const int length = seq < p.cache.seqs ? cached_length(p.cache.lengths[seq], p.cache.table_width, 1 << p.cache.page_shift) : 0;
  return p.count && length ? p.count << p.cache.page_shift : length;
}
template <typename MATCH>
__device__ __forceinline__ bool paged_find(const PagedAttentionParams& p, MATCH match, PagedItem& item) {
  const int lane = lane_id(), seqs = p.cache.seqs;
  int total = 0, tiles = 0;
  for (int s0 = 0; s0 < seqs; s0 += kWave) {
    tiles = paged_tiles(paged_tokens(p, s0 + lane));
    total += tiles;
  }
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) total += __shfl_xor(total, d);
  item.part_tiles = paged_part_tiles(uniform(total), p.slots, kPagedLeast);
  int before = 0;
  for (int s0 = 0; s0 < seqs; s0 += kWave) {
    if (seqs > kWave) tiles = paged_tiles(paged_tokens(p, s0 + lane));
    const int parts = s0 + lane < seqs ? paged_parts(tiles, item.part_tiles) : 0;
    int upto = parts;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
      const int other = __shfl_up(upto, d);
      if (lane >= d) upto += other;
    }
    const unsigned long long hit = __ballot(match(s0 + lane, before + upto - parts, parts));
    if (hit) {
      const int at = __ffsll(hit) - 1;
      item.seq = s0 + at;
      item.parts = uniform(__shfl(parts, at));
      item.first_item = uniform(__shfl(before + upto - parts, at));
      return true;
    }
    before += uniform(__shfl(upto, kWave - 1));
  }
  return false;
}

// Two e4m3 codes of a dword to a pair of 16-bit values (exact).
template <bool BF16, bool HIGH>
__device__ __forceinline__ unsigned widen_pair(unsigned codes) {
  if constexpr (BF16) return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, 1.f, HIGH));
  else return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, 1.f, HIGH));
}

template <bool BF16, int D, bool E8>
__global__ __launch_bounds__(kPagedWaves * 64, D == 256 && !E8 ? 1 : 2) void paged_attention_kernel(PagedAttentionParams p) {
  typedef unsigned short u16;
  constexpr int ES = E8 ? 1 : 2;               // bytes of an element
  constexpr int KS = D / 32;                   // steps of the sum over features
  constexpr int KW = D * ES / 64;              // 16-byte loads of a lane for the keys of 16 tokens (E8: each is two steps)
  constexpr int F = D / 16;                    // features of a value row that a lane has: operands of the second product
  constexpr int VD = F * ES / 4;               // ... in dwords: 1 .. 8
  constexpr bool PV_BF16 = BF16 || E8;         // (an e4m3 value's power of two goes to the probability, which fp16 has not the range for)
  extern __shared__ __align__(16) float smem[];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int col = lane & 15, g = lane >> 4;
  const int kv_head = blockIdx.y / p.group_tiles, group_tile = blockIdx.y % p.group_tiles;
  const int rows = min(16, p.group - group_tile * 16);   // queries
  const PagedParams& cache = p.cache;

  PagedItem item;
  const int id = blockIdx.x;
  if (!paged_find(p, [&](int, int first, int parts) { return first + parts > id; }, item)) return;
  item.part = id - item.first_item;
  const int seq = item.seq;
  const int length = cached_length(cache.lengths[seq], cache.table_width, 1 << cache.page_shift);
  const int tokens = p.count && length ? p.count << cache.page_shift : length;
  const long long part_tokens = (long long)item.part_tiles * kPagedTile;
  const int begin = (int)min((long long)tokens, item.part * part_tokens), end = (int)min((long long)tokens, (item.part + 1) * part_tokens);

  // ---- queries: columns of the first product ----
  u32x4 fq[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) fq[s] = u32x4{0u, 0u, 0u, 0u};
  if (col < rows) {
    const u16* q = p.q + seq * p.q_strides[0] + (long long)(kv_head * p.group + group_tile * 16 + col) * p.q_strides[1];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d = E8 ? s / 2 * 64 + g * 16 + s % 2 * 8 : s * 32 + g * 8;
      unsigned w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = q[(d + 2 * j) * p.q_strides[2]] | (unsigned)q[(d + 2 * j + 1) * p.q_strides[2]] << 16;
      fq[s] = u32x4{w[0], w[1], w[2], w[3]};
    }
  }

  // ---- the pages of the part: 64 entries of the table (or list) in the lanes ----
  const int* table = cache.table + (size_t)seq * cache.table_row;
  const int* listed = p.count ? p.listed + ((size_t)seq * cache.kv_heads + kv_head) * p.count : nullptr;
  const int entries = p.count ? p.count : cache.table_width;
  int window = -(1 << 30), entry_logical = 0, entry_page = -1;
  auto look_up = [&](int entry) {
    window = entry;
    const int e = entry + lane;
    entry_page = -1, entry_logical = 0;
    if (e < entries) {
      entry_logical = listed ? listed[e] : e;
      if ((unsigned)entry_logical < (unsigned)cache.table_width) entry_page = table[entry_logical];
      else entry_logical = 0;
    }
  };

  struct Tile {
    u32x4 k[2][KW];
    unsigned v[2][4][VD];
    unsigned ke[2], ve[2];   // exponents of this lane's four tokens
    int valid[2];
  };
  auto load = [&](int t, Tile& tile) {
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      const PagedPlace place = paged_place(t + a * 16, cache.page_shift);
      if (place.entry >= window + kWave || place.entry < window) look_up(place.entry);
      const int page = __builtin_amdgcn_readlane(entry_page, place.entry - window), logical = __builtin_amdgcn_readlane(entry_logical, place.entry - window);
      const int valid = place.entry < entries ? paged_valid(logical, place.slot, cache.page_shift, page, cache.pages, length) : 0;
      tile.valid[a] = valid;
      if (valid == 0) {
#pragma unroll
        for (int s = 0; s < KW; ++s) tile.k[a][s] = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int d = 0; d < VD; ++d) tile.v[a][i][d] = 0u;
        tile.ke[a] = tile.ve[a] = 0x7F7F7F7Fu;
        continue;
      }
      const size_t row0 = ((size_t)kv_head << cache.page_shift) + place.slot;
      const unsigned char* k = static_cast<const unsigned char*>(cache.keys) + ((long long)page * cache.key_page + (long long)row0 * D) * ES;
      const unsigned char* v = static_cast<const unsigned char*>(cache.values) + ((long long)page * cache.value_page + (long long)row0 * D) * ES;
#pragma unroll
      for (int s = 0; s < KW; ++s) tile.k[a][s] = *reinterpret_cast<const u32x4*>(k + col * (D * ES) + s * 64 + g * 16);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned char* at = v + (g * 4 + i) * (D * ES);
        // (heads of 256 in 16 bits: two halves of 128, so that a load of 16 lanes is 256 consecutive bytes)
        if constexpr (VD == 8) {
          *reinterpret_cast<u32x4*>(&tile.v[a][i][0]) = *reinterpret_cast<const u32x4*>(at + col * 16);
          *reinterpret_cast<u32x4*>(&tile.v[a][i][4]) = *reinterpret_cast<const u32x4*>(at + 256 + col * 16);
        } else if constexpr (VD == 4) {
          *reinterpret_cast<u32x4*>(&tile.v[a][i][0]) = *reinterpret_cast<const u32x4*>(at + col * 16);
        } else if constexpr (VD == 2) {
          *reinterpret_cast<u32x2*>(&tile.v[a][i][0]) = *reinterpret_cast<const u32x2*>(at + col * 8);
        } else {
          tile.v[a][i][0] = *reinterpret_cast<const unsigned*>(at + col * 4);
        }
      }
      if constexpr (E8) {
        const size_t at = (((size_t)page * cache.kv_heads) << cache.page_shift) + row0 + g * 4;
        tile.ke[a] = *reinterpret_cast<const unsigned*>(cache.key_exponents + at);
        tile.ve[a] = *reinterpret_cast<const unsigned*>(cache.value_exponents + at);
      }
    }
  };

  f32x4 o[F];
#pragma unroll
  for (int j = 0; j < F; ++j) o[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  float top = -INFINITY, sum = 0.f;   // of this lane's query: the maximum so far (all groups'), this group's share of the sum
  int attended = 0;

  auto compute = [&](Tile& tile) {
    attended += tile.valid[0] + tile.valid[1];
    f32x4 s[2];
#pragma unroll
    for (int a = 0; a < 2; ++a) s[a] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < KS; ++e)
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        u32x4 fk;
        if constexpr (E8) {
          const unsigned c0 = tile.k[a][e / 2][e % 2 * 2], c1 = tile.k[a][e / 2][e % 2 * 2 + 1];
          fk = u32x4{widen_pair<BF16, false>(c0), widen_pair<BF16, true>(c0), widen_pair<BF16, false>(c1), widen_pair<BF16, true>(c1)};
        } else {
          fk = tile.k[a][e];
        }
        s[a] = mfma_16x16x32<BF16>(fk, fq[e], s[a]);
      }
    if constexpr (E8) {
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[a][r] *= power_of_two(tile.ke[a] >> (r * 8) & 0xFFu);
    }
    if (tile.valid[0] + tile.valid[1] != 32) {   // (uniform) tokens that are not attended to leave no trace, infinities and NaN included
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (g * 4 + r >= tile.valid[a]) {
            s[a][r] = -INFINITY;
#pragma unroll
            for (int d = 0; d < VD; ++d) tile.v[a][r][d] = 0u;
            if constexpr (E8) tile.ve[a] = (tile.ve[a] & ~(0xFFu << (r * 8))) | 0x7Fu << (r * 8);
          }
    }
    float m = s[0][0];
#pragma unroll
    for (int a = 0; a < 2; ++a)
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
    const float shift = top == -INFINITY ? 0.f : -top * p.scale_log2;
    u32x4 hi, lo;
#pragma unroll
    for (int a = 0; a < 2; ++a) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[a][r] = __builtin_amdgcn_exp2f(fmaf(s[a][r], p.scale_log2, shift));   // (exp2(-infinity) = 0)
        sum += s[a][r];
        if constexpr (E8) s[a][r] *= power_of_two(tile.ve[a] >> (r * 8) & 0xFFu);
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        hi[a * 2 + r] = pack_pair<PV_BF16>(s[a][2 * r], s[a][2 * r + 1]);
        float h0, h1;
        unpack_pair<PV_BF16>(hi[a * 2 + r], h0, h1);
        lo[a * 2 + r] = pack_pair<PV_BF16>(s[a][2 * r] - h0, s[a][2 * r + 1] - h1);
      }
    }
#pragma unroll
    for (int j = 0; j < F; ++j) {
      u32x4 fv;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int a = w / 2, r = w % 2 * 2;   // tokens r and r + 1 of the four in subtile a
        if constexpr (E8) {
          // byte j of both rows side by side, then widened
          const unsigned pair = __builtin_amdgcn_perm(tile.v[a][r + 1][j / 4], tile.v[a][r][j / 4], (j % 4) | (4 + j % 4) << 8);
          fv[w] = widen_pair<PV_BF16, false>(pair);
        } else {
          fv[w] = __builtin_amdgcn_perm(tile.v[a][r + 1][j / 2], tile.v[a][r][j / 2], j % 2 ? 0x07060302u : 0x05040100u);
        }
      }
      o[j] = mfma_16x16x32<PV_BF16>(fv, hi, o[j]);
      o[j] = mfma_16x16x32<PV_BF16>(fv, lo, o[j]);
    }
  };

  // ---- the part's tiles, a wavefront's in turn, the next one's loads ahead of the present one's products ----
  Tile one, two;
  int t = begin + wave * 32;
  constexpr int STEP = kPagedWaves * 32;
  if (t < end) load(t, one);
  while (t < end) {
    if (t + STEP < end) load(t + STEP, two);
    compute(one);
    t += STEP;
    if (t >= end) break;
    if (t + STEP < end) load(t + STEP, one);
    compute(two);
    t += STEP;
  }

  // ---- the wavefronts meet ----
  sum += __shfl_xor(sum, 16);
  sum += __shfl_xor(sum, 32);
  if (attended == 0) sum = -1.f;   // no token at all: zeros, whatever the formula says of an empty sum
  float* sums = smem;                                  // [wave][row][D]
  float* tops = smem + kPagedWaves * rows * D;         // [wave][row] (maximum, sum)
  if (col < rows) {
    float* mine = sums + (wave * rows + col) * D;
#pragma unroll
    for (int j = 0; j < F; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int c = g * 4 + r;   // the lane column whose features these are
        const int d = VD == 8 ? j / 8 * 128 + c * 8 + j % 8 : c * F + j;
        mine[d] = o[j][r];
      }
    if (g == 0) tops[(wave * rows + col) * 2] = top, tops[(wave * rows + col) * 2 + 1] = sum;
  }
  __syncthreads();
  const bool whole = item.parts == 1;
  const size_t result = (size_t)blockIdx.y * gridDim.x + blockIdx.x;
  for (int i = threadIdx.x; i < rows * D; i += kPagedWaves * 64) {
    const int row = i / D, d = i % D;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < kPagedWaves; ++w) m = fmaxf(m, tops[(w * rows + row) * 2]);
    float total = 0.f, acc = 0.f;
    bool any = false;
#pragma unroll
    for (int w = 0; w < kPagedWaves; ++w) {
      const float mine = tops[(w * rows + row) * 2], part = tops[(w * rows + row) * 2 + 1];
      if (part == -1.f) continue;
      any = true;
      const float keep = mine == m ? 1.f : __builtin_amdgcn_exp2f((mine - m) * p.scale_log2);
      total += keep * part;
      acc += keep * sums[(w * rows + row) * D + d];
    }
    if (whole) {
      const int head = kv_head * p.group + group_tile * 16 + row;
      p.out[seq * p.out_strides[0] + head * p.out_strides[1] + d * p.out_strides[2]] = f32_to_16(any ? acc / total : 0.f, BF16);
    } else {
      p.partial[(result * p.pitch + row) * D + d] = acc;
      if (d == 0) p.stats[(result * p.pitch + row) * 2] = m, p.stats[(result * p.pitch + row) * 2 + 1] = any ? total : -1.f;
    }
  }
}

// Parts of a sequence into its result, a workgroup per sequence and query head: 256 / (D / 4) parts side by side, a thread four
// features with a running maximum; they meet in LDS.
template <bool BF16, int D>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttentionParams p, int items) {
  constexpr int LANES = D / 4, SIDE = 256 / LANES;   // threads of a row; parts side by side
  __shared__ float4 accs[SIDE][LANES];
  __shared__ float tops[SIDE][2];
  const int seq = blockIdx.x, head = blockIdx.y;
  const int kv_head = head / p.group, in_group = head % p.group;
  PagedItem item;
  if (!paged_find(p, [&](int s, int, int) { return s == seq; }, item)) return;
  if (item.parts == 1) return;
  const int lane = threadIdx.x % LANES, side = threadIdx.x / LANES;
  const size_t y = (size_t)kv_head * p.group_tiles + in_group / 16, row = in_group % 16;
  float4 acc = {0.f, 0.f, 0.f, 0.f};
  float top = -INFINITY, sum = -1.f;
  for (int i = side; i < item.parts; i += SIDE) {
    const size_t result = (y * items + item.first_item + i) * p.pitch + row;
    const float m = p.stats[result * 2], part = p.stats[result * 2 + 1];
    const float4 x = *reinterpret_cast<const float4*>(p.partial + result * D + lane * 4);
    if (part == -1.f) continue;
    const float now = fmaxf(top, m);
    const float keep = top == now ? 1.f : __builtin_amdgcn_exp2f((top - now) * p.scale_log2), in = m == now ? 1.f : __builtin_amdgcn_exp2f((m - now) * p.scale_log2);
    sum = (sum == -1.f ? 0.f : sum * keep) + part * in;
    acc.x = acc.x * keep + x.x * in, acc.y = acc.y * keep + x.y * in, acc.z = acc.z * keep + x.z * in, acc.w = acc.w * keep + x.w * in;
    top = now;
  }
  accs[side][lane] = acc;
  if (lane == 0) tops[side][0] = top, tops[side][1] = sum;
  __syncthreads();
  if (threadIdx.x >= D) return;
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < SIDE; ++i) m = fmaxf(m, tops[i][0]);
  float total = 0.f, x = 0.f;
  bool any = false;
#pragma unroll
  for (int i = 0; i < SIDE; ++i) {
    if (tops[i][1] == -1.f) continue;
    any = true;
    const float keep = tops[i][0] == m ? 1.f : __builtin_amdgcn_exp2f((tops[i][0] - m) * p.scale_log2);
    total += keep * tops[i][1];
    x += keep * reinterpret_cast<const float*>(accs[i])[threadIdx.x];
  }
  p.out[seq * p.out_strides[0] + head * p.out_strides[1] + threadIdx.x * p.out_strides[2]] = f32_to_16(any ? x / total : 0.f, BF16);
}

}  // namespace iex
