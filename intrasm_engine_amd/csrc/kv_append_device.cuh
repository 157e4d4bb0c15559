// New tokens' keys and values into a paged cache, with the position rotation of keys and queries on the way.
//
// A token at position t has its features rotated in r / 2 planes, plane j by the angle a(t, j) whose cosine and sine are given:
//   y0 = x0 cos - x1 sin,   y1 = x1 cos + x0 sin
// where (x0, x1) are features (j, j + r/2) or, interleaved, (2j, 2j + 1).  Products and sums are rounded one by one in 32 bits (no
// fused multiply-add), so that anybody's plain formula gives the same bits before the one rounding to the cache's type.
//
// A workgroup has the new tokens of one sequence in one span of positions (whole pages) for a few heads of one kind: keys,
// queries or values.  A thread has a unit of 16 features of a token: both halves of eight planes, so a rotation needs nobody
// else.  An 8-bit row (e4m3) takes the least power of two as its scale that brings its largest magnitude to 448: scaling by it
// is exact, so the rounding to e4m3 is the only one.  Bounds (smallest and largest stored key per page and feature) are written
// by the one workgroup that has a page's new tokens, from LDS; a page that had tokens before keeps theirs.
//
// What bounds it: prompts by memory (each feature is read and written once), a step of generation by latency: lengths -> table
// -> store is the longest chain of loads.  Measured: 16 prompts of 512 tokens, 3 x 32 heads of 128, feature-major 79 us = 5.1 TB/s read
// and written; 23 of 3 .. 5001 tokens, 32 + 2 x 8 heads, into e4m3 with bounds 96 us = 4.2 (waiting for a row's maximum, vector
// units 36 %); a step of one sequence of 3 x 32 heads 3.0 us, of 64 of 32 + 2 x 8 heads with bounds 4.2.
#pragma once
#include "paged_cache_device.cuh"

namespace iex {

struct AppendOperand {
  const unsigned short* x;
  long long per_token, per_head, per_feature;   // strides
};

struct AppendParams {
  PagedParams cache;
  int tokens, heads, rotary, columns, per_group;   // heads of a workgroup (keys: one, where there are bounds)
  const int* offsets;                     // null: one token per sequence (kv_append_step_kernel)
  AppendOperand k, q, v;
  unsigned short* q_out;
  long long out_token, out_head, out_feature;   // strides
  const float* rotation;
  unsigned short* bounds;
};

// Largest of LANES consecutive lanes, LANES in {4, 8, 16}, in every one of them.
template <int LANES>
__device__ __forceinline__ unsigned group_max(unsigned v) {
  auto with = [&](unsigned w) { v = v > w ? v : w; };
  with((unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, true));
  with((unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, true));
  if (LANES >= 8) with((unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, true));
  if (LANES >= 16) with((unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xf, 0xf, true));
  return v;
}

// One plane.
__device__ __forceinline__ void rotate(float& a, float& b, float c, float s) {
#pragma clang fp contract(off)
  const float ac = a * c, bs = b * s, bc = b * c, as = a * s;
  a = ac - bs;
  b = bc + as;
}

// What a workgroup has: rows low .. high of the span of positions from `begin` on, token `first_token` + row of the call; heads
// head0 .. head_end of one kind.
struct AppendWork {
  Appended a;
  int seq, begin, low, high, first_token;
  bool is_k, is_q;
  int head0, head_end;
  const unsigned short* src;
  long long per_token, per_head, per_feature;   // its strides
};
__device__ __forceinline__ void take_operand(const AppendParams& p, AppendWork& w) {
  // (bit by bit: chosen by address the arguments would be copied to memory)
  auto of_kind = [&](long long k, long long q, long long v) { return w.is_k ? k : w.is_q ? q : v; };
  w.src = reinterpret_cast<const unsigned short*>(of_kind((long long)p.k.x, (long long)p.q.x, (long long)p.v.x));
  w.per_token = of_kind(p.k.per_token, p.q.per_token, p.v.per_token);
  w.per_head = of_kind(p.k.per_head, p.q.per_head, p.v.per_head);
  w.per_feature = of_kind(p.k.per_feature, p.q.per_feature, p.v.per_feature);
}
__device__ __forceinline__ bool append_work(const AppendParams& p, AppendWork& w) {
  const PagedParams& cache = p.cache;
  const int lane = lane_id(), span = append_span(1 << cache.page_shift), most = cache.table_width << cache.page_shift;
  int in_seq = 0;
  int before = 0;
  bool found = false;
  for (int s0 = 0; s0 <= cache.seqs && !found; s0 += kWave) {   // (every wavefront on its own; nearly always one step)
    const int s = s0 + lane;
    const int begin = s <= cache.seqs ? p.offsets[s] : 0, end = s < cache.seqs ? p.offsets[s + 1] : 0;
    const Appended mine = appended(s, cache.seqs, p.tokens, begin, end, s < cache.seqs ? cache.lengths[s] : 0, most);
    const int spans = append_spans(mine, span), upto = wave_scan(spans);
    const unsigned long long past = __ballot(before + upto > (int)blockIdx.x);
    if (past) {
      const int at = __ffsll(past) - 1;
      w.seq = s0 + at;
      w.a = Appended{bcast_i(mine.first, at), bcast_i(mine.count, at), bcast_i(mine.position, at), bcast_i(mine.sound, at) != 0};
      in_seq = blockIdx.x - (before + bcast_i(upto - spans, at));
      found = true;
    }
    before += bcast_i(upto, kWave - 1);
  }
  if (!found) return false;
  w.begin = (w.a.position / span + in_seq) * span;
  w.low = w.a.position > w.begin ? w.a.position - w.begin : 0;
  const int end = w.a.position + w.a.count - w.begin;
  w.high = end < span ? end : span;
  w.first_token = w.a.first + w.begin - w.a.position;

  const int k_groups = p.bounds ? cache.kv_heads : (cache.kv_heads + p.per_group - 1) / p.per_group;
  const int q_groups = (p.heads + p.per_group - 1) / p.per_group;
  int group = blockIdx.y;
  w.is_k = group < k_groups, w.is_q = !w.is_k && group < k_groups + q_groups;
  const int per = w.is_k && p.bounds ? 1 : p.per_group;
  group -= w.is_k ? 0 : w.is_q ? k_groups : k_groups + q_groups;
  w.head0 = group * per, w.head_end = min(w.head0 + per, w.is_q ? p.heads : cache.kv_heads);
  take_operand(p, w);
  return w.a.sound || w.is_q;
}

// A thread's unit of a row: its two chunks of eight features, and the cosines and sines of its planes.
struct UnitPlace {
  bool turned;
  int c0, c1;
  __device__ __forceinline__ UnitPlace(const AppendParams& p, const AppendWork& w, int u, bool interleaved) {
    turned = (w.is_k || w.is_q) && u < p.rotary / 16 && w.a.sound;
    c0 = !interleaved && turned ? u : 2 * u, c1 = !interleaved && turned ? u + p.rotary / 16 : 2 * u + 1;
  }
};
struct Planes {
  float4 c[2], s[2];
  __device__ __forceinline__ void load(const AppendParams& p, int position, int u) {
    const float4* t = reinterpret_cast<const float4*>(p.rotation + (size_t)position * p.rotary + 8 * u);
    c[0] = t[0], c[1] = t[1], s[0] = t[p.rotary / 8], s[1] = t[p.rotary / 8 + 1];
  }
};
// The unit's 16 features in 32 bits and, turned, in 16.
template <bool BF16, bool INTERLEAVED>
__device__ __forceinline__ void turn_unit(bool turned, const Planes& t, u32x4& raw0, u32x4& raw1, float (&x)[16]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    unpack_pair<BF16>(raw0[j], x[2 * j], x[2 * j + 1]);
    unpack_pair<BF16>(raw1[j], x[8 + 2 * j], x[9 + 2 * j]);
  }
  if (!turned) return;
  const float c[8] = {t.c[0].x, t.c[0].y, t.c[0].z, t.c[0].w, t.c[1].x, t.c[1].y, t.c[1].z, t.c[1].w};
  const float s[8] = {t.s[0].x, t.s[0].y, t.s[0].z, t.s[0].w, t.s[1].x, t.s[1].y, t.s[1].z, t.s[1].w};
#pragma unroll
  for (int i = 0; i < 8; ++i) rotate(x[INTERLEAVED ? 2 * i : i], x[INTERLEAVED ? 2 * i + 1 : 8 + i], c[i], s[i]);
#pragma unroll
  for (int j = 0; j < 4; ++j) raw0[j] = pack_pair<BF16>(x[2 * j], x[2 * j + 1]), raw1[j] = pack_pair<BF16>(x[8 + 2 * j], x[9 + 2 * j]);
}

// A unit of a key's or value's row into its page (all lanes of the row together: an 8-bit row's exponent is of all of it).  x becomes
// what was stored.
template <bool BF16, int D, bool E8>
__device__ __forceinline__ void store_unit(const AppendParams& p, bool is_k, int page, int head, int slot, int u, const UnitPlace& at, const u32x4& raw0, const u32x4& raw1,
                                           float (&x)[16]) {
  const PagedParams& cache = p.cache;
  const bool kept = (unsigned)page < (unsigned)cache.pages;
  const size_t in_page = ((size_t)head << cache.page_shift) + slot;   // rows before it in its page
  const long long page_at = (long long)page * (is_k ? cache.key_page : cache.value_page);
  if constexpr (E8) {
    unsigned top = 0;
#pragma unroll
    for (int j = 0; j < 16; ++j) top = max(top, __float_as_uint(x[j]) & 0x7FFFFFFFu);
    top = group_max<D / 16>(top);
    const bool finite = top < 0x7F800000u;
    if (__ballot(!finite)) {   // an infinity or NaN in some row: the exponent is of the largest finite magnitude, so that the others are kept
      unsigned rest = 0;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const unsigned magnitude = __float_as_uint(x[j]) & 0x7FFFFFFFu;
        rest = max(rest, magnitude < 0x7F800000u ? magnitude : 0u);
      }
      top = group_max<D / 16>(rest);
    }
    const int e = e4m3_exponent(top);
    const float down = power_of_two(254 - e), up = power_of_two(e);
    unsigned code[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      code[j] = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * j] * down, x[4 * j + 1] * down, 0, false);
      code[j] = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * j + 2] * down, x[4 * j + 3] * down, code[j], true);
    }
    if (!finite) {   // e4m3 has no infinity: it becomes NaN too
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if ((__float_as_uint(x[j]) & 0x7FFFFFFFu) >= 0x7F800000u) code[j / 4] |= 0x7Fu << (j % 4 * 8);
    }
    if (kept) {
      unsigned char* to = static_cast<unsigned char*>(const_cast<void*>(is_k ? cache.keys : cache.values)) + page_at + in_page * D;
      *reinterpret_cast<u32x2*>(to + at.c0 * 8) = u32x2{code[0], code[1]};
      *reinterpret_cast<u32x2*>(to + at.c1 * 8) = u32x2{code[2], code[3]};
      if (u == 0)
        const_cast<unsigned char*>(is_k ? cache.key_exponents : cache.value_exponents)[(((size_t)page * cache.kv_heads) << cache.page_shift) + in_page] = (unsigned char)e;
    }
    if (is_k && p.bounds) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        typedef float f2 __attribute__((ext_vector_type(2)));
        const f2 two = j % 2 ? __builtin_amdgcn_cvt_pk_f32_fp8(code[j / 2], true) : __builtin_amdgcn_cvt_pk_f32_fp8(code[j / 2], false);
        unpack_pair<BF16>(pack_pair<BF16>(two.x * up, two.y * up), x[2 * j], x[2 * j + 1]);
      }
    }
  } else {
    if (kept) {
      unsigned short* to = static_cast<unsigned short*>(const_cast<void*>(is_k ? cache.keys : cache.values)) + page_at + in_page * D;
      *reinterpret_cast<u32x4*>(to + at.c0 * 8) = raw0;
      *reinterpret_cast<u32x4*>(to + at.c1 * 8) = raw1;
    }
    if (is_k && p.bounds) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        unpack_pair<BF16>(raw0[j], x[2 * j], x[2 * j + 1]);
        unpack_pair<BF16>(raw1[j], x[8 + 2 * j], x[9 + 2 * j]);
      }
    }
  }
}

// Bounds of the pages that a span's new tokens are in, from rows of what was stored, in LDS.  A thread has a feature and a side (0
// smallest, 1 largest), two of them for heads of 256.  Only the page of the sequence's first new token can have had tokens before.
template <bool BF16, int D>
struct AppendBounds {
  static constexpr int SIDES = 2 * D > 256 ? 2 * D / 256 : 1;
  float extreme[SIDES];
  __device__ __forceinline__ void begin(const AppendParams& p, const AppendWork& w) {
    const PagedParams& cache = p.cache;
#pragma unroll
    for (int e = 0; e < SIDES; ++e) extreme[e] = (threadIdx.x + e * 256) / D == 0 ? INFINITY : -INFINITY;
    if ((w.a.position & ((1 << cache.page_shift) - 1)) == 0 || w.a.position < w.begin) return;
    const int page = cache.table[(size_t)w.seq * cache.table_row + (w.a.position >> cache.page_shift)];
    if ((unsigned)page >= (unsigned)cache.pages) return;
#pragma unroll
    for (int e = 0; e < SIDES; ++e)
      if (threadIdx.x + e * 256 < 2 * D) extreme[e] = f32_of_16<BF16>(p.bounds[((size_t)page * cache.kv_heads + w.head0) * (2 * D) + threadIdx.x + e * 256]);
  }
  // Rows first .. last of the span, stored[] from row `base` on.
  __device__ __forceinline__ void add(const AppendParams& p, const AppendWork& w, const float* stored, int base, int first, int last) {
    const PagedParams& cache = p.cache;
#pragma unroll
    for (int e = 0; e < SIDES; ++e) {
      const int f = (threadIdx.x + e * 256) % D, side = (threadIdx.x + e * 256) / D;
      if (side > 1) continue;
      for (int i = first; i < last; ++i) {
        const float x = stored[(i - base) * D + f];
        extreme[e] = side ? larger(extreme[e], x) : smaller(extreme[e], x);
        const int at = w.begin + i;
        if (i + 1 != w.high && ((at + 1) & ((1 << cache.page_shift) - 1)) != 0) continue;
        // the page's last new token
        const int page = cache.table[(size_t)w.seq * cache.table_row + (at >> cache.page_shift)];
        if ((unsigned)page < (unsigned)cache.pages)
          p.bounds[(((size_t)page * cache.kv_heads + w.head0) * 2 + side) * D + f] = (unsigned short)pack_pair<BF16>(extreme[e], 0.f);
        extreme[e] = side ? -INFINITY : INFINITY;
      }
    }
  }
};
__device__ __forceinline__ void stored_unit(float* row, const UnitPlace& at, const float (&x)[16]) {
#pragma unroll
  for (int j = 0; j < 8; j += 4) {
    *reinterpret_cast<float4*>(row + at.c0 * 8 + j) = float4{x[j], x[j + 1], x[j + 2], x[j + 3]};
    *reinterpret_cast<float4*>(row + at.c1 * 8 + j) = float4{x[8 + j], x[9 + j], x[10 + j], x[11 + j]};
  }
}

// One token per sequence, a step of generation: rows are sequences, each with a place of its own, so a page's bounds are its row's
// business.  STAGED: operands of any strides, lanes along the sequences, through LDS.
template <bool BF16, int D, bool E8, bool INTERLEAVED, bool STAGED>
__global__ __launch_bounds__(256, 4) void kv_append_step_kernel(AppendParams p) {
  typedef unsigned short u16;
  constexpr int U = D / 16, R = 256 / U;
  __shared__ __align__(16) u16 tile[STAGED ? R * D : 8];
  auto chunk_at = [&](int t, int c) { return reinterpret_cast<u32x4*>(tile + t * D + (c ^ (t & 7)) * 8); };
  const PagedParams& cache = p.cache;
  const int u = threadIdx.x % U, r = threadIdx.x / U, first = blockIdx.x * R, seq = first + r;
  const bool mine = seq < p.tokens;
  AppendWork w;
  int head = blockIdx.y;
  w.is_k = head < cache.kv_heads, w.is_q = !w.is_k && head < cache.kv_heads + p.heads;
  head -= w.is_k ? 0 : w.is_q ? cache.kv_heads : cache.kv_heads + p.heads;
  take_operand(p, w);
  const u16* src = w.src + head * w.per_head;
  w.a = mine ? appended(seq, cache.seqs, p.tokens, seq, seq + 1, cache.lengths[seq], cache.table_width << cache.page_shift) : Appended{0, 0, 0, 0};
  const UnitPlace at(p, w, u, INTERLEAVED);
  u32x4 raw0 = {0u, 0u, 0u, 0u}, raw1 = raw0;
  if constexpr (STAGED) {
    for (int i = threadIdx.x; i < R * (D / 8); i += 256) {
      const int t = i % R, chunk = i / R;
      if (first + t >= p.tokens) continue;
      const u16* x = src + (long long)(first + t) * w.per_token + chunk * 8 * w.per_feature;
      u16 e[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] = x[j * w.per_feature];
      u32x4 packed;
#pragma unroll
      for (int j = 0; j < 4; ++j) packed[j] = e[2 * j] | (unsigned)e[2 * j + 1] << 16;
      *chunk_at(t, chunk) = packed;
    }
  } else if (mine) {
    const u16* from = src + (long long)seq * w.per_token;
    raw0 = *reinterpret_cast<const u32x4*>(from + at.c0 * 8);
    raw1 = *reinterpret_cast<const u32x4*>(from + at.c1 * 8);
  }
  Planes planes;
  if (at.turned) planes.load(p, w.a.position, u);   // (of a sound row)
  const int slot = w.a.position & ((1 << cache.page_shift) - 1);
  int page = -1;
  if (!w.is_q && w.a.sound) page = cache.table[(size_t)seq * cache.table_row + (w.a.position >> cache.page_shift)];
  const bool bounded = w.is_k && p.bounds && (unsigned)page < (unsigned)cache.pages;
  u16* const bounds = bounded ? p.bounds + ((size_t)page * cache.kv_heads + head) * (2 * D) : nullptr;
  u32x4 old[2][2];   // smallest, largest
  if (bounded && slot != 0) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      old[i][0] = *reinterpret_cast<const u32x4*>(bounds + i * D + at.c0 * 8);
      old[i][1] = *reinterpret_cast<const u32x4*>(bounds + i * D + at.c1 * 8);
    }
  }
  if constexpr (STAGED) {
    __syncthreads();
    if (mine) raw0 = *chunk_at(r, at.c0), raw1 = *chunk_at(r, at.c1);
  }
  float x[16];
  turn_unit<BF16, INTERLEAVED>(at.turned, planes, raw0, raw1, x);
  if (w.is_q) {
    if (!w.a.sound) raw0 = raw1 = u32x4{0u, 0u, 0u, 0u};
    u16* out = p.q_out + head * p.out_head;
    if constexpr (STAGED) {
      if (mine) *chunk_at(r, at.c0) = raw0, *chunk_at(r, at.c1) = raw1;
      __syncthreads();
      for (int i = threadIdx.x; i < R * (D / 8); i += 256) {
        const int t = i % R, chunk = i / R;
        if (first + t >= p.tokens) continue;
        const u32x4 packed = *chunk_at(t, chunk);
        u16* to = out + (long long)(first + t) * p.out_token + chunk * 8 * p.out_feature;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          to[2 * j * p.out_feature] = (u16)packed[j];
          to[(2 * j + 1) * p.out_feature] = (u16)(packed[j] >> 16);
        }
      }
    } else if (mine) {
      *reinterpret_cast<u32x4*>(out + (long long)seq * p.out_token + at.c0 * 8) = raw0;
      *reinterpret_cast<u32x4*>(out + (long long)seq * p.out_token + at.c1 * 8) = raw1;
    }
    return;
  }
  store_unit<BF16, D, E8>(p, w.is_k, page, head, slot, u, at, raw0, raw1, x);
  if (!bounded) return;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    u32x4 now[2];
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float a = x[c * 8 + 2 * j], b = x[c * 8 + 2 * j + 1];
        if (slot != 0) {
          float a0, b0;
          unpack_pair<BF16>(old[i][c][j], a0, b0);
          a = i ? larger(a0, a) : smaller(a0, a), b = i ? larger(b0, b) : smaller(b0, b);
        }
        now[c][j] = pack_pair<BF16>(a, b);
      }
    *reinterpret_cast<u32x4*>(bounds + i * D + at.c0 * 8) = now[0];
    *reinterpret_cast<u32x4*>(bounds + i * D + at.c1 * 8) = now[1];
  }
}

// Operands whose rows are whole aligned 16-byte chunks.  HEADS: heads whose loads are in flight at once.
template <bool BF16, int D, bool E8, bool INTERLEAVED, int HEADS>
__global__ __launch_bounds__(256, 4) void kv_append_kernel(AppendParams p) {
  constexpr int U = D / 16, R = 256 / U;   // units of a row, rows of a step
  extern __shared__ __align__(16) unsigned char smem[];
  float* const stored = reinterpret_cast<float*>(smem);   // bounds: R x D
  AppendWork w;
  if (!append_work(p, w)) return;
  const int u = threadIdx.x % U, r = threadIdx.x / U, page_size = 1 << p.cache.page_shift;
  const UnitPlace at(p, w, u, INTERLEAVED);
  const bool bounded = w.is_k && p.bounds;   // (head0 is the only head)
  AppendBounds<BF16, D> bounds;
  bool begun = false;

  for (int block = w.low / R * R; block < w.high; block += R) {
    const int row = block + r, position = w.begin + row;
    const bool mine = row >= w.low && row < w.high;
    Planes planes;
    if (at.turned && mine) planes.load(p, position, u);
    int page = -1;
    if (!w.is_q && mine) page = p.cache.table[(size_t)w.seq * p.cache.table_row + (position >> p.cache.page_shift)];
    for (int head1 = w.head0; head1 < w.head_end; head1 += HEADS) {
      u32x4 raw[HEADS][2];
#pragma unroll
      for (int h = 0; h < HEADS; ++h) {
        raw[h][0] = raw[h][1] = u32x4{0u, 0u, 0u, 0u};
        if (!mine || head1 + h >= w.head_end) continue;
        const unsigned short* from = w.src + (long long)(w.first_token + row) * w.per_token + (head1 + h) * w.per_head;
        raw[h][0] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(from + at.c0 * 8));
        raw[h][1] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(from + at.c1 * 8));
      }
      if (bounded && !begun) bounds.begin(p, w), begun = true;   // (two loads one behind the other, beside the rows')
#pragma unroll
      for (int h = 0; h < HEADS; ++h) {
        const int head = head1 + h;
        if (head >= w.head_end) break;
        float x[16];
        turn_unit<BF16, INTERLEAVED>(at.turned && mine, planes, raw[h][0], raw[h][1], x);
        if (w.is_q) {
          if (!mine) continue;
          if (!w.a.sound) raw[h][0] = raw[h][1] = u32x4{0u, 0u, 0u, 0u};
          unsigned short* to = p.q_out + (long long)(w.first_token + row) * p.out_token + head * p.out_head;
          *reinterpret_cast<u32x4*>(to + at.c0 * 8) = raw[h][0];
          *reinterpret_cast<u32x4*>(to + at.c1 * 8) = raw[h][1];
          continue;
        }
        store_unit<BF16, D, E8>(p, w.is_k, page, head, position & (page_size - 1), u, at, raw[h][0], raw[h][1], x);
        if (bounded) {
          __syncthreads();   // the step before has been read
          if (mine) stored_unit(stored + r * D, at, x);
          __syncthreads();
          bounds.add(p, w, stored, block, max(w.low, block), min(w.high, block + R));
        }
      }
    }
  }
}

// Operands of any strides, by tiles of 64 tokens x D features of a head through LDS (rows of tokens, chunk c of token t at c ^ (t / 8
// % 8)).  Where tokens are next to each other (features x tokens, as a projection W @ X leaves them: p.columns) they are read and
// written 16 bytes at a time, eight tokens of a feature, and turned around two bytes at a time in LDS; else two bytes at a time in memory.
constexpr int kColumnTokens = 64;
typedef u32x4 AnyChunk __attribute__((aligned(2)));
template <bool BF16, int D, bool E8, bool INTERLEAVED>
__global__ __launch_bounds__(256, 4) void kv_append_columns_kernel(AppendParams p) {
  typedef unsigned short u16;
  constexpr int U = D / 16, R = 256 / U, T = kColumnTokens;
  extern __shared__ __align__(16) unsigned char smem[];
  u16* const tile = reinterpret_cast<u16*>(smem);                        // T x D
  float* const stored = reinterpret_cast<float*>(smem + T * D * 2);      // bounds: R x D
  auto element = [&](int t, int f) -> u16* { return tile + (t * D + ((f / 8) ^ (t / 8 % 8)) * 8 + f % 8); };
  AppendWork w;
  if (!append_work(p, w)) return;
  const int u = threadIdx.x % U, r = threadIdx.x / U, page_size = 1 << p.cache.page_shift;
  const UnitPlace at(p, w, u, INTERLEAVED);
  const bool bounded = w.is_k && p.bounds;
  AppendBounds<BF16, D> bounds;
  if (bounded) bounds.begin(p, w);

  for (int block = w.low / T * T; block < w.high; block += T) {
    const int low = max(w.low, block) - block, high = min(w.high, block + T) - block;   // rows of the tile
    const int token0 = w.first_token + block;                                           // ... of row 0
    // 64 tokens in eight chunks of eight, from any token on: sequences that begin off a chunk 16 x 511 tokens of 3 x 32 heads of 128 152 ->
    // 126 us, but 3 x 1001 of 32 + 2 x 8 heads of 256 52 -> 64
    const bool whole = low == 0 && high == T && (D < 256 || token0 % 8 == 0);
    for (int head = w.head0; head < w.head_end; ++head) {
      const u16* src = w.src + head * w.per_head;
      __syncthreads();   // the tile before has been read
      if (p.columns && whole) {
        constexpr int LOADS = T * D / 8 / 256;
        const int c = threadIdx.x % 8, f = threadIdx.x / 8;
        u32x4 x[LOADS];
#pragma unroll
        for (int k = 0; k < LOADS; ++k) x[k] = __builtin_nontemporal_load(reinterpret_cast<const AnyChunk*>(src + (f + k * 32) * w.per_feature + token0 + c * 8));
#pragma unroll
        for (int k = 0; k < LOADS; ++k) {
          u16* to = element(c * 8, f + k * 32);
#pragma unroll
          for (int j = 0; j < 8; ++j) to[j * D] = (u16)(x[k][j / 2] >> (j % 2 * 16));
        }
      } else if (p.columns) {
        const int from = (token0 + low) / 8 * 8, chunks = (token0 + high - from + 7) / 8;   // (up to nine hold the rows)
        for (int i = threadIdx.x; i < chunks * D; i += 256) {
          const int f = i / chunks, token = from + i % chunks * 8;
          u16 e[8];
          if (token + 8 <= p.tokens) {
            const u32x4 x = *reinterpret_cast<const u32x4*>(src + f * w.per_feature + token);
#pragma unroll
            for (int j = 0; j < 8; ++j) e[j] = (u16)(x[j / 2] >> (j % 2 * 16));
          } else {   // the operand's last tokens
#pragma unroll
            for (int j = 0; j < 8; ++j) e[j] = token + j < p.tokens ? src[f * w.per_feature + token + j] : 0;
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int t = token + j - token0;
            if (t >= low && t < high) *element(t, f) = e[j];
          }
        }
      } else {
        for (int i = threadIdx.x; i < T * (D / 8); i += 256) {
          const int t = i % T, chunk = i / T;
          if (t < low || t >= high) continue;
          const u16* x = src + (long long)(token0 + t) * w.per_token + chunk * 8 * w.per_feature;
          u16 e[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) e[j] = x[j * w.per_feature];
          u32x4 packed;
#pragma unroll
          for (int j = 0; j < 4; ++j) packed[j] = e[2 * j] | (unsigned)e[2 * j + 1] << 16;
          *reinterpret_cast<u32x4*>(element(t, chunk * 8)) = packed;
        }
      }
      __syncthreads();
#pragma unroll 1
      for (int sub = low / R * R; sub < high; sub += R) {
        const int t = sub + r, position = w.begin + block + t;
        const bool mine = t >= low && t < high;
        Planes planes;
        if (at.turned && mine) planes.load(p, position, u);
        int page = -1;
        if (!w.is_q && mine) page = p.cache.table[(size_t)w.seq * p.cache.table_row + (position >> p.cache.page_shift)];
        u32x4 raw0 = {0u, 0u, 0u, 0u}, raw1 = raw0;
        if (mine) raw0 = *reinterpret_cast<const u32x4*>(element(t, at.c0 * 8)), raw1 = *reinterpret_cast<const u32x4*>(element(t, at.c1 * 8));
        float x[16];
        turn_unit<BF16, INTERLEAVED>(at.turned && mine, planes, raw0, raw1, x);
        if (w.is_q) {
          if (!w.a.sound) raw0 = raw1 = u32x4{0u, 0u, 0u, 0u};
          if (mine) *reinterpret_cast<u32x4*>(element(t, at.c0 * 8)) = raw0, *reinterpret_cast<u32x4*>(element(t, at.c1 * 8)) = raw1;
          continue;
        }
        store_unit<BF16, D, E8>(p, w.is_k, page, head, position & (page_size - 1), u, at, raw0, raw1, x);
        if (bounded) {
          __syncthreads();   // the step before has been read
          if (mine) stored_unit(stored + r * D, at, x);
          __syncthreads();
          bounds.add(p, w, stored, block + sub, block + max(low, sub), block + min(high, sub + R));
        }
      }
      if (!w.is_q) continue;
      __syncthreads();
      u16* out = p.q_out + head * p.out_head;
      if (p.columns && whole) {
        constexpr int STORES = T * D / 8 / 256;
        const int c = threadIdx.x % 8, f = threadIdx.x / 8;
#pragma unroll
        for (int k = 0; k < STORES; ++k) {
          const u16* x = element(c * 8, f + k * 32);
          u32x4 packed;
#pragma unroll
          for (int j = 0; j < 4; ++j) packed[j] = x[2 * j * D] | (unsigned)x[(2 * j + 1) * D] << 16;
          *reinterpret_cast<AnyChunk*>(out + (f + k * 32) * p.out_feature + token0 + c * 8) = packed;
        }
      } else if (p.columns) {
        for (int i = threadIdx.x; i < T * D; i += 256) {
          const int t = i % T, f = i / T;
          if (t >= low && t < high) out[f * p.out_feature + token0 + t] = *element(t, f);
        }
      } else {
        for (int i = threadIdx.x; i < T * (D / 8); i += 256) {
          const int t = i % T, chunk = i / T;
          if (t < low || t >= high) continue;
          const u32x4 packed = *reinterpret_cast<const u32x4*>(element(t, chunk * 8));
          u16* to = out + (long long)(token0 + t) * p.out_token + chunk * 8 * p.out_feature;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            to[2 * j * p.out_feature] = (u16)packed[j];
            to[(2 * j + 1) * p.out_feature] = (u16)(packed[j] >> 16);
          }
        }
      }
    }
  }
}

}  // namespace iex
