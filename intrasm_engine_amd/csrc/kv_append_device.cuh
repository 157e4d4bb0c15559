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
// -> store is the longest chain of loads.
#pragma once
#include "paged_cache_device.cuh"

namespace iex {

struct AppendParams {
  PagedParams cache;
  int tokens, heads, rotary, per_group;   // heads of a workgroup (keys: one, where there are bounds)
  const int* offsets;                     // null: one token per sequence
  const unsigned short* k;
  const unsigned short* v;
  const unsigned short* q;
  unsigned short* q_out;
  long long k_strides[3], v_strides[3], q_strides[3], out_strides[3];   // token, head, feature
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

// Eight planes: x[first(i)], x[second(i)].
template <bool INTERLEAVED>
__device__ __forceinline__ void rotate_unit(float (&x)[16], const float (&c)[8], const float (&s)[8]) {
#pragma clang fp contract(off)
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float& a = x[INTERLEAVED ? 2 * i : i];
    float& b = x[INTERLEAVED ? 2 * i + 1 : i + 8];
    const float ac = a * c[i], bs = b * s[i], bc = b * c[i], as = a * s[i];
    a = ac - bs;
    b = bc + as;
  }
}

template <bool BF16, int D, bool E8, bool STAGED, bool INTERLEAVED>
__global__ __launch_bounds__(256) void kv_append_kernel(AppendParams p) {
  typedef unsigned short u16;
  constexpr int U = D / 16, R = 256 / U;   // units of a row, rows of a step
  __shared__ __align__(16) u16 tile[STAGED ? R * D : 8];
  __shared__ __align__(16) float stored[R * D];
  const PagedParams& cache = p.cache;
  const int tid = threadIdx.x, lane = tid & 63;
  const int page_size = 1 << cache.page_shift, span = append_span(page_size), most = cache.table_width << cache.page_shift;

  // ---- whose tokens ----
  Appended a;
  int seq, in_seq = 0;
  if (!p.offsets) {
    seq = blockIdx.x;
    a = appended(seq, cache.seqs, p.tokens, seq, seq + 1, cache.lengths[seq], most);
  } else {
    int before = 0;
    bool found = false;
    for (int s0 = 0; s0 <= cache.seqs && !found; s0 += kWave) {   // (every wavefront on its own; nearly always one step)
      const int s = s0 + lane;
      const int begin = s <= cache.seqs ? p.offsets[s] : 0, end = s < cache.seqs ? p.offsets[s + 1] : 0;
      const Appended mine = appended(s, cache.seqs, p.tokens, begin, end, s < cache.seqs ? cache.lengths[s] : 0, most);
      const int spans = append_spans(mine, span);
      int upto = spans;
#pragma unroll
      for (int d = 1; d < kWave; d <<= 1) {
        const int other = __shfl_up(upto, d);
        if (lane >= d) upto += other;
      }
      const unsigned long long past = __ballot(before + upto > (int)blockIdx.x);
      if (past) {
        const int at = __ffsll((unsigned long long)past) - 1;
        seq = s0 + at;
        a.first = __shfl(mine.first, at), a.count = __shfl(mine.count, at), a.position = __shfl(mine.position, at);
        a.sound = __shfl((int)mine.sound, at);
        in_seq = blockIdx.x - (before + __shfl(upto - spans, at));
        found = true;
      }
      before += __shfl(upto, kWave - 1);
    }
    if (!found) return;
  }
  const int begin = (a.position / span + in_seq) * span;   // first position of the span
  const int low = a.position > begin ? a.position - begin : 0;
  const int end = a.position + a.count - begin, high = end < span ? end : span;   // rows low .. high of it are new tokens

  // ---- which heads, of what ----
  const int k_groups = p.bounds ? cache.kv_heads : (cache.kv_heads + p.per_group - 1) / p.per_group;
  const int q_groups = (p.heads + p.per_group - 1) / p.per_group;
  int group = blockIdx.y;
  const bool is_k = group < k_groups, is_q = !is_k && group < k_groups + q_groups;
  const int per = is_k && p.bounds ? 1 : p.per_group;
  group -= is_k ? 0 : is_q ? k_groups : k_groups + q_groups;
  const int head0 = group * per, head_end = min(head0 + per, is_q ? p.heads : cache.kv_heads);
  if (!a.sound && !is_q) return;
  const u16* src = is_k ? p.k : is_q ? p.q : p.v;
  const long long* st = is_k ? p.k_strides : is_q ? p.q_strides : p.v_strides;

  const int u = tid % U, r = tid / U;
  const bool turned = (is_k || is_q) && u < p.rotary / 16;
  const int c0 = !INTERLEAVED && turned ? u : 2 * u, c1 = !INTERLEAVED && turned ? u + p.rotary / 16 : 2 * u + 1;

  // bounds: this thread's feature and side (0 smallest, 1 largest), two of them for heads of 256
  constexpr int SIDES = 2 * D > 256 ? 2 * D / 256 : 1;
  float extreme[SIDES];
#pragma unroll
  for (int e = 0; e < SIDES; ++e) extreme[e] = (tid + e * 256) / D == 0 ? INFINITY : -INFINITY;

  for (int block = low / R * R; block < high; block += R) {
    const int row = block + r, position = begin + row;
    const bool mine = row >= low && row < high;
    const int token = a.first + position - a.position;
    float c[8], s[8];
    if (turned && mine && a.sound) {
      const float4* t = reinterpret_cast<const float4*>(p.rotation + (size_t)position * p.rotary + 8 * u);
      const float4* t2 = t + p.rotary / 8;
      const float4 a0 = t[0], a1 = t[1], b0 = t2[0], b1 = t2[1];
      c[0] = a0.x, c[1] = a0.y, c[2] = a0.z, c[3] = a0.w, c[4] = a1.x, c[5] = a1.y, c[6] = a1.z, c[7] = a1.w;
      s[0] = b0.x, s[1] = b0.y, s[2] = b0.z, s[3] = b0.w, s[4] = b1.x, s[5] = b1.y, s[6] = b1.z, s[7] = b1.w;
    }
    int page = -1;
    const int slot = position & (page_size - 1);
    if (!is_q && mine) page = cache.table[(size_t)seq * cache.table_row + (position >> cache.page_shift)];
    const bool kept = (unsigned)page < (unsigned)cache.pages;

    for (int head = head0; head < head_end; ++head) {
      // ---- 16 features ----
      u32x4 raw0 = {0u, 0u, 0u, 0u}, raw1 = {0u, 0u, 0u, 0u};
      if constexpr (STAGED) {   // any strides: lanes along the tokens, through LDS
        __syncthreads();
        for (int i = tid; i < R * (D / 8); i += 256) {
          const int t = i % R, chunk = i / R, at = block + t;
          if (at < low || at >= high) continue;
          const u16* from = src + (long long)(a.first + begin + at - a.position) * st[0] + head * st[1] + chunk * 8 * st[2];
          unsigned w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) w[j] = from[2 * j * st[2]] | (unsigned)from[(2 * j + 1) * st[2]] << 16;
          *reinterpret_cast<u32x4*>(&tile[t * D + (chunk ^ (t & 7)) * 8]) = u32x4{w[0], w[1], w[2], w[3]};
        }
        __syncthreads();
        if (mine) {
          raw0 = *reinterpret_cast<const u32x4*>(&tile[r * D + (c0 ^ (r & 7)) * 8]);
          raw1 = *reinterpret_cast<const u32x4*>(&tile[r * D + (c1 ^ (r & 7)) * 8]);
        }
      } else if (mine) {
        const u16* from = src + (long long)token * st[0] + head * st[1];
        raw0 = *reinterpret_cast<const u32x4*>(from + c0 * 8);
        raw1 = *reinterpret_cast<const u32x4*>(from + c1 * 8);
      }
      float x[16];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        unpack_pair<BF16>(raw0[j], x[2 * j], x[2 * j + 1]);
        unpack_pair<BF16>(raw1[j], x[8 + 2 * j], x[9 + 2 * j]);
      }
      if (turned && mine && a.sound) {
        rotate_unit<INTERLEAVED>(x, c, s);
#pragma unroll
        for (int j = 0; j < 4; ++j) raw0[j] = pack_pair<BF16>(x[2 * j], x[2 * j + 1]), raw1[j] = pack_pair<BF16>(x[8 + 2 * j], x[9 + 2 * j]);
      }

      if (is_q) {
        if (!a.sound) raw0 = raw1 = u32x4{0u, 0u, 0u, 0u};
        if constexpr (STAGED) {
          if (mine) {
            *reinterpret_cast<u32x4*>(&tile[r * D + (c0 ^ (r & 7)) * 8]) = raw0;
            *reinterpret_cast<u32x4*>(&tile[r * D + (c1 ^ (r & 7)) * 8]) = raw1;
          }
          __syncthreads();
          for (int i = tid; i < R * (D / 8); i += 256) {
            const int t = i % R, chunk = i / R, at = block + t;
            if (at < low || at >= high) continue;
            const u32x4 w = *reinterpret_cast<const u32x4*>(&tile[t * D + (chunk ^ (t & 7)) * 8]);
            u16* to = p.q_out + (long long)(a.first + begin + at - a.position) * p.out_strides[0] + head * p.out_strides[1] + chunk * 8 * p.out_strides[2];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              to[2 * j * p.out_strides[2]] = (u16)w[j];
              to[(2 * j + 1) * p.out_strides[2]] = (u16)(w[j] >> 16);
            }
          }
        } else if (mine) {
          u16* to = p.q_out + (long long)token * p.out_strides[0] + head * p.out_strides[1];
          *reinterpret_cast<u32x4*>(to + c0 * 8) = raw0;
          *reinterpret_cast<u32x4*>(to + c1 * 8) = raw1;
        }
        continue;
      }

      // ---- into the cache ----
      const size_t in_page = ((size_t)head << cache.page_shift) + slot;   // rows before it in its page
      const long long page_at = (long long)page * (is_k ? cache.key_page : cache.value_page);
      if constexpr (E8) {
        unsigned top = 0;
#pragma unroll
        for (int j = 0; j < 16; ++j) top = max(top, __float_as_uint(x[j]) & 0x7FFFFFFFu);
        top = group_max<U>(top);
        const int e = e4m3_exponent(top);
        const float down = power_of_two(254 - e), up = power_of_two(e);
        unsigned code[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          code[j] = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * j] * down, x[4 * j + 1] * down, 0, false);
          code[j] = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * j + 2] * down, x[4 * j + 3] * down, code[j], true);
        }
        if (top >= 0x7F800000u) {   // an infinity or NaN in the row: e4m3 has no infinity, both become its NaN
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if ((__float_as_uint(x[j]) & 0x7FFFFFFFu) >= 0x7F800000u) code[j / 4] |= 0x7Fu << (j % 4 * 8);
        }
        if (kept) {
          unsigned char* to = static_cast<unsigned char*>(const_cast<void*>(is_k ? cache.keys : cache.values)) + page_at + in_page * D;
          *reinterpret_cast<u32x2*>(to + c0 * 8) = u32x2{code[0], code[1]};
          *reinterpret_cast<u32x2*>(to + c1 * 8) = u32x2{code[2], code[3]};
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
          u16* to = static_cast<u16*>(const_cast<void*>(is_k ? cache.keys : cache.values)) + page_at + in_page * D;
          *reinterpret_cast<u32x4*>(to + c0 * 8) = raw0;
          *reinterpret_cast<u32x4*>(to + c1 * 8) = raw1;
        }
        if (is_k && p.bounds) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            unpack_pair<BF16>(raw0[j], x[2 * j], x[2 * j + 1]);
            unpack_pair<BF16>(raw1[j], x[8 + 2 * j], x[9 + 2 * j]);
          }
        }
      }

      if (is_k && p.bounds) {   // (head0 is the only one)
        __syncthreads();   // the step before has been read
        if (mine) {
#pragma unroll
          for (int j = 0; j < 8; j += 4) {
            *reinterpret_cast<float4*>(&stored[r * D + c0 * 8 + j]) = float4{x[j], x[j + 1], x[j + 2], x[j + 3]};
            *reinterpret_cast<float4*>(&stored[r * D + c1 * 8 + j]) = float4{x[8 + j], x[9 + j], x[10 + j], x[11 + j]};
          }
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < SIDES; ++e) {
          const int f = (tid + e * 256) % D, side = (tid + e * 256) / D;
          if (side > 1) continue;
          const int last = min(high, block + R);
          for (int i = max(low, block); i < last; ++i) {
            const float x1 = stored[(i - block) * D + f];
            extreme[e] = side ? larger(extreme[e], x1) : smaller(extreme[e], x1);
            const int at = begin + i;
            if (i + 1 != high && ((at + 1) & (page_size - 1)) != 0) continue;
            // the page's last new token
            const int logical = at >> cache.page_shift, to_page = cache.table[(size_t)seq * cache.table_row + logical];
            if ((unsigned)to_page < (unsigned)cache.pages) {
              u16* b = p.bounds + (((size_t)to_page * cache.kv_heads + head) * 2 + side) * D + f;
              if (a.position > logical << cache.page_shift) {
                const float old = f32_of_16<BF16>(*b);
                extreme[e] = side ? larger(extreme[e], old) : smaller(extreme[e], old);
              }
              *b = (u16)pack_pair<BF16>(extreme[e], 0.f);
            }
            extreme[e] = side ? -INFINITY : INFINITY;
          }
        }
      }
    }
  }
}

}  // namespace iex
