// The launches of appending to a paged cache (kv_append_device.cuh), with positions given (AT) or not: a source file each.
#pragma once
#include "kv_append_device.cuh"
#include "paged_cache_host.h"

namespace iex {

int launch_kv_append(const iex_paged_cache& c, const AppendParams& p, bool rows, bool interleaved, hipStream_t s);
int launch_kv_append_at(const iex_paged_cache& c, const AppendParams& p, bool rows, bool interleaved, hipStream_t s);

namespace {

template <bool BF16, int D, bool E8, bool INTERLEAVED, bool AT>
int launch(const AppendParams& p, bool rows, hipStream_t s) {
  const char* type = BF16 ? "bf16" : "f16";
  const char* stored = E8 ? "e4m3" : "16";
  constexpr int per_step = 256 / (D / 16);   // rows of 256 threads
  const int kv_heads = p.cache.kv_heads, kv_groups = ceil_div(kv_heads, p.per_group);
  if (!p.offsets) {
    note_kernel("kv_append_step_kernel<%s, %d, %s, %s>%s", type, D, stored, rows ? "rows" : "staged", AT ? " (positions given)" : "");
    const dim3 grid(ceil_div(p.tokens, per_step), 2 * kv_heads + p.heads);
    if (rows) hipLaunchKernelGGL((kv_append_step_kernel<BF16, D, E8, INTERLEAVED, AT, false>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((kv_append_step_kernel<BF16, D, E8, INTERLEAVED, AT, true>), grid, dim3(256), 0, s, p);
    return check_hip(hipGetLastError(), "kv_append launch");
  }
  const dim3 grid((unsigned)append_most_spans(p.tokens, p.cache.seqs, append_span(1 << p.cache.page_shift)),
                  (p.bounds ? kv_heads : kv_groups) + kv_groups + ceil_div(p.heads, p.per_group));
  const int lds = (rows ? 0 : kColumnTokens * D * 2) + (p.bounds ? per_step * D * 4 : 0);
  note_kernel("%s<%s, %d, %s> (%d heads a workgroup)%s", rows ? "kv_append_kernel" : "kv_append_columns_kernel", type, D, stored, p.per_group, AT ? " (positions given)" : "");
  if (!rows) hipLaunchKernelGGL((kv_append_columns_kernel<BF16, D, E8, INTERLEAVED, AT>), grid, dim3(256), lds, s, p);
  else if (p.per_group == 1) hipLaunchKernelGGL((kv_append_kernel<BF16, D, E8, INTERLEAVED, AT, 1>), grid, dim3(256), lds, s, p);
  else hipLaunchKernelGGL((kv_append_kernel<BF16, D, E8, INTERLEAVED, AT, 4>), grid, dim3(256), lds, s, p);
  return check_hip(hipGetLastError(), "kv_append launch");
}

template <bool BF16, int D, bool E8, bool AT>
int launch_forms(const AppendParams& p, bool rows, bool interleaved, hipStream_t s) {
  return interleaved ? launch<BF16, D, E8, true, AT>(p, rows, s) : launch<BF16, D, E8, false, AT>(p, rows, s);
}

template <bool BF16, bool AT>
int launch_type(const AppendParams& p, int head_dim, bool e8, bool rows, bool interleaved, hipStream_t s) {
  if (head_dim == 64) return e8 ? launch_forms<BF16, 64, true, AT>(p, rows, interleaved, s) : launch_forms<BF16, 64, false, AT>(p, rows, interleaved, s);
  if (head_dim == 128) return e8 ? launch_forms<BF16, 128, true, AT>(p, rows, interleaved, s) : launch_forms<BF16, 128, false, AT>(p, rows, interleaved, s);
  return e8 ? launch_forms<BF16, 256, true, AT>(p, rows, interleaved, s) : launch_forms<BF16, 256, false, AT>(p, rows, interleaved, s);
}

template <bool AT>
int launch_append(const iex_paged_cache& c, const AppendParams& p, bool rows, bool interleaved, hipStream_t s) {
  return c.dtype == IEX_BF16 ? launch_type<true, AT>(p, c.head_dim, c.eight_bits, rows, interleaved, s) : launch_type<false, AT>(p, c.head_dim, c.eight_bits, rows, interleaved, s);
}

}  // namespace
}  // namespace iex
