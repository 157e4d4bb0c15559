// Appending to a paged cache with positions given (kv_append_device.cuh).
#include "kv_append_host.h"

namespace iex {

int launch_kv_append_at(const iex_paged_cache& c, const AppendParams& p, bool rows, bool interleaved, hipStream_t s) { return launch_append<true>(c, p, rows, interleaved, s); }

}  // namespace iex
