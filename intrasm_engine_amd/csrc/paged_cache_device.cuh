// What the kernels of the paged cache share on the device.
#pragma once
#include "gemm_device.cuh"
#include "paged_cache.h"

namespace iex {

struct PagedParams {
  int pages, page_shift, kv_heads, seqs, table_width;
  long long key_page, value_page, table_row;   // strides in elements
  const void* keys;
  const void* values;
  const unsigned char* key_exponents;
  const unsigned char* value_exponents;
  const int* table;
  const int* lengths;
};

__device__ __forceinline__ float power_of_two(int biased) { return __uint_as_float((unsigned)biased << 23); }

// Sums of lanes 0 .. this one; the last lane's is the total.
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);   // row_shr 1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);   // row_bcast 15, 31
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
  return v;
}

// An element of either 16-bit type in 32 bits.
template <bool BF16>
__device__ __forceinline__ float f32_of_16(unsigned short bits) {
  if constexpr (BF16) return __uint_as_float((unsigned)bits << 16);
  else return (float)__builtin_bit_cast(_Float16, bits);
}
template <bool BF16>
__device__ __forceinline__ void unpack_pair(unsigned two, float& a, float& b) {
  a = f32_of_16<BF16>((unsigned short)two);
  if constexpr (BF16) b = __uint_as_float(two & 0xFFFF0000u);
  else b = f32_of_16<BF16>((unsigned short)(two >> 16));
}

// The smaller / larger of two, NaN if either is.
__device__ __forceinline__ float smaller(float a, float b) { return a < b || a != a ? a : b; }
__device__ __forceinline__ float larger(float a, float b) { return a > b || a != a ? a : b; }

}  // namespace iex
