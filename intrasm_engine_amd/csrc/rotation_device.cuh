// Rotation of features by positions.  A token has its features rotated in r / 2 planes, plane j by an angle whose cosine and sine stand in a table, one row
// a position:
//   y0 = x0 cos - x1 sin,   y1 = x1 cos + x0 sin
// where (x0, x1) are features (j, j + r/2) or, interleaved, (2j, 2j + 1).  Products and sums are rounded one by one in 32 bits (no
// fused multiply-add), so that anybody's plain formula gives the same bits before the one rounding to the result's type.
//
// A position can have up to four axes (time, height, width ..): plane j's row is then the position on its axis.
#pragma once
#include "paged_cache_device.cuh"

namespace iex {

struct Rotation {
  const float* table;     // (rows, features): cosines, then sines
  int rows, features;     // features that turn
  const int* positions;   // (axes, tokens); null: where a token lies is its position (AT below)
  long long axis_stride;
  int axes;
  unsigned long long axis_of[4];   // two bits a plane
};

// Plane numbers of an axis each (32 planes a word), by the words' own registers.
__device__ __forceinline__ unsigned long long axis_word(const Rotation& r, int word) {
  return word == 0 ? r.axis_of[0] : word == 1 ? r.axis_of[1] : word == 2 ? r.axis_of[2] : r.axis_of[3];
}

// The table's row of a token on an axis.  A position below zero counts as zero, one behind the table has no cosine (NaN).
struct RotationRow {
  int row;
  bool known;
  __device__ __forceinline__ RotationRow(const Rotation& r, int position) : row(max(0, min(position, r.rows - 1))), known(position < r.rows) {}
};
// A token's positions on all axes.
struct RotationPlace {
  int at[4];
  __device__ __forceinline__ RotationPlace(const Rotation& r, int token) {
    at[0] = r.positions[token];
#pragma unroll
    for (int a = 1; a < 4; ++a) at[a] = a < r.axes ? r.positions[a * r.axis_stride + token] : 0;
  }
  __device__ __forceinline__ int on(int axis) const { return axis == 0 ? at[0] : axis == 1 ? at[1] : axis == 2 ? at[2] : at[3]; }
};

// One plane.
__device__ __forceinline__ void rotate(float& a, float& b, float c, float s) {
#pragma clang fp contract(off)
  const float ac = a * c, bs = b * s, bc = b * c, as = a * s;
  a = ac - bs;
  b = bc + as;
}

// Cosine and sine of one plane.
__device__ __forceinline__ int axis_of(const Rotation& r, int plane) { return r.axes > 1 ? (int)(axis_word(r, plane / 32) >> (plane % 32 * 2)) & 3 : 0; }
__device__ __forceinline__ void load_plane_at(const Rotation& r, int position, int plane, float& c, float& s) {
  const RotationRow row(r, position);
  const float* t = r.table + (size_t)row.row * r.features + plane;
  c = t[0], s = t[r.features / 2];
  if (!row.known) c = s = NAN;
}
__device__ __forceinline__ void load_plane(const Rotation& r, int token, int plane, float& c, float& s) {
  load_plane_at(r, r.positions[axis_of(r, plane) * r.axis_stride + token], plane, c, s);
}

// ... of planes 8 u .. 8 u + 7, 16 bytes at a time where they are of one axis.
struct Planes {
  float c[8], s[8];
  __device__ __forceinline__ void load_row(const Rotation& r, int row, int u) {
    const float4* t = reinterpret_cast<const float4*>(r.table + (size_t)row * r.features + 8 * u);
    const float4 four[4] = {t[0], t[1], t[r.features / 8], t[r.features / 8 + 1]};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      c[4 * i] = four[i].x, c[4 * i + 1] = four[i].y, c[4 * i + 2] = four[i].z, c[4 * i + 3] = four[i].w;
      s[4 * i] = four[2 + i].x, s[4 * i + 1] = four[2 + i].y, s[4 * i + 2] = four[2 + i].z, s[4 * i + 3] = four[2 + i].w;
    }
  }
  // AT: by the token's given positions; else its place in its sequence, which the table has.
  template <bool AT>
  __device__ __forceinline__ void load(const Rotation& r, int token, int where, int u) {
    if constexpr (!AT) {
      load_row(r, where, u);
    } else {
      const RotationPlace place(r, token);
      const unsigned axes = r.axes > 1 ? (unsigned)(axis_word(r, u / 4) >> (u % 4 * 16)) & 0xFFFFu : 0u;
      if (__ballot(axes != (axes & 3u) * 0x5555u)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) load_plane_at(r, place.on(axes >> (2 * i) & 3u), 8 * u + i, c[i], s[i]);
        return;
      }
      const RotationRow row(r, place.on(axes & 3u));
      load_row(r, row.row, u);
      if (!row.known) {
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = s[i] = NAN;
      }
    }
  }
};

}  // namespace iex
