// Rotation of features by positions on one to four axes, and its gradient, the same rotation the other way (rotation_device.cuh has the formula).
//
// What bounds it: memory, every feature is read and written once, 2 r more words of the table a token.  So a thread keeps its planes' cosines and
// sines in registers for several heads, and loads and stores are 16 bytes or more:
//   rows      features next to each other: a thread has eight planes of a token, 16 features
//   columns   tokens next to each other (features x tokens, as a projection W @ X leaves them): a thread has a plane of eight tokens, or, where they
//             are not 16-byte aligned, planes of a token
//   single    everything else: a thread has a plane of a token
// Measured: 30001 tokens of 32 heads of 128 in bf16, 64 features by three axes in turn, rows 114 us = 4.4 TB/s read and written (with streaming loads 123, with
// streaming stores 133); 8192 tokens in fp16, columns 30 us = 4.6; 300 tokens of 16 heads of 64 4.1.  In fp32, 30001 tokens of 32 heads of 128, forward or back:
// rows 215 us = 4.6 TB/s, columns (30000 tokens) 229 = 4.3, tokens at other alignments 312 = 3.2.
#include "rotation_host.h"

namespace iex {
namespace {

struct RotateParams {
  Rotation rotation;
  int tokens, heads, dim, back, per_thread, planes;   // heads that a thread takes one after the other; planes of a workgroup (tokens)
  const void* x;
  void* out;
  long long x_strides[3], out_strides[3];   // token, head, feature
};

// Eight elements next to each other, 16-byte aligned, and in 32 bits.
template <int DTYPE> struct rotate_element { typedef unsigned short type; };
template <> struct rotate_element<IEX_F32> { typedef float type; };
template <int DTYPE>
__device__ __forceinline__ float widen(typename rotate_element<DTYPE>::type x) {
  if constexpr (DTYPE == IEX_F32) return x;
  else return f32_of_16<DTYPE == IEX_BF16>(x);
}
template <int DTYPE>
__device__ __forceinline__ typename rotate_element<DTYPE>::type narrow(float x) {
  if constexpr (DTYPE == IEX_F32) return x;
  else return (unsigned short)pack_pair<DTYPE == IEX_BF16>(x, 0.f);
}
template <int DTYPE>
struct Eight {
  typedef typename rotate_element<DTYPE>::type T;
  static constexpr int N = DTYPE == IEX_F32 ? 2 : 1;
  u32x4 raw[N];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < N; ++i) raw[i] = *(reinterpret_cast<const u32x4*>(p) + i);
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < N; ++i) *(reinterpret_cast<u32x4*>(p) + i) = raw[i];
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DTYPE == IEX_F32) x[2 * i] = __uint_as_float(raw[i / 2][i % 2 * 2]), x[2 * i + 1] = __uint_as_float(raw[i / 2][i % 2 * 2 + 1]);
      else unpack_pair<DTYPE == IEX_BF16>(raw[0][i], x[2 * i], x[2 * i + 1]);
    }
  }
  __device__ __forceinline__ void set(const float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DTYPE == IEX_F32) raw[i / 2][i % 2 * 2] = __float_as_uint(x[2 * i]), raw[i / 2][i % 2 * 2 + 1] = __float_as_uint(x[2 * i + 1]);
      else raw[0][i] = pack_pair<DTYPE == IEX_BF16>(x[2 * i], x[2 * i + 1]);
    }
  }
};

// Heads whose loads are in flight at once: of rows (eight: 300 tokens of 16 heads of 64 5.0 us, 4.1 by four), of columns (four: 8192 tokens of 32 heads of
// 128 37.7, 34.0 by eight).
constexpr int kRowsAhead = 4, kColumnsAhead = 8;

template <int DTYPE, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rotate_rows_kernel(RotateParams p) {
  typedef typename rotate_element<DTYPE>::type T;
  typedef Eight<DTYPE> Chunk;
  const int units = p.dim / 16, turned_units = p.rotation.features / 16;
  const long long item = (long long)blockIdx.x * 256 + threadIdx.x;
  const int token = (int)(item / units), u = (int)(item % units);
  if (token >= p.tokens) return;
  const bool turned = u < turned_units;
  const int c0 = turned && !INTERLEAVED ? u : 2 * u, c1 = turned && !INTERLEAVED ? u + turned_units : 2 * u + 1;   // chunks of eight features
  Planes planes;
  if (turned) {
    planes.load<true>(p.rotation, token, 0, u);
    if (p.back) {
#pragma unroll
      for (int i = 0; i < 8; ++i) planes.s[i] = -planes.s[i];
    }
  }
  const T* x = static_cast<const T*>(p.x) + token * p.x_strides[0];
  T* out = static_cast<T*>(p.out) + token * p.out_strides[0];
  const int first = blockIdx.y * p.per_thread, end = min(p.heads, first + p.per_thread);
  for (int head = first; head < end; head += kRowsAhead) {
    Chunk a[kRowsAhead], b[kRowsAhead];
#pragma unroll
    for (int h = 0; h < kRowsAhead; ++h) {
      if (head + h >= end) break;
      a[h].load(x + (head + h) * p.x_strides[1] + c0 * 8);
      b[h].load(x + (head + h) * p.x_strides[1] + c1 * 8);
    }
#pragma unroll
    for (int h = 0; h < kRowsAhead; ++h) {
      if (head + h >= end) break;
      if (turned) {
        float f[16];
        a[h].get(reinterpret_cast<float(&)[8]>(f[0]));
        b[h].get(reinterpret_cast<float(&)[8]>(f[8]));
#pragma unroll
        for (int i = 0; i < 8; ++i) rotate(f[INTERLEAVED ? 2 * i : i], f[INTERLEAVED ? 2 * i + 1 : 8 + i], planes.c[i], planes.s[i]);
        a[h].set(reinterpret_cast<const float(&)[8]>(f[0]));
        b[h].set(reinterpret_cast<const float(&)[8]>(f[8]));
      }
      a[h].store(out + (head + h) * p.out_strides[1] + c0 * 8);
      b[h].store(out + (head + h) * p.out_strides[1] + c1 * 8);
    }
  }
}

// A plane's two features: of a turned plane, or of the features behind (dim - features is even).
__device__ __forceinline__ void pair_of(const RotateParams& p, int plane, bool interleaved, int& f0, int& f1) {
  const int half = p.rotation.features / 2;
  f0 = plane < half && !interleaved ? plane : 2 * plane, f1 = plane < half && !interleaved ? plane + half : 2 * plane + 1;
}

// Cosines and sines of 64 tokens and up to 32 planes, by a workgroup into LDS: the table's rows are read where they are long and used where tokens are next
// to each other.  (Each lane its own from memory: 7394 tokens of 16 heads of 256 74 us, 39 so.)
constexpr int kTilePlanes = 32, kTilePitch = 65;   // (without bank conflicts where it is read; writes are two lanes a bank, by fewer planes up to eight)
struct RotationTile {
  float c[kTilePlanes][kTilePitch], s[kTilePlanes][kTilePitch];
  __device__ __forceinline__ void load(const RotateParams& p, int token0, int plane0, int planes) {   // a power of two
    const int turned = p.rotation.features / 2;
    for (int i = threadIdx.x; i < 64 * planes; i += 256) {
      const int plane = i & (planes - 1), token = i / planes;
      if (token0 + token >= p.tokens || plane0 + plane >= turned) continue;
      float its, other;
      load_plane(p.rotation, token0 + token, plane0 + plane, its, other);
      c[plane][token] = its, s[plane][token] = p.back ? -other : other;
    }
    __syncthreads();
  }
};

// Workgroups of 64 tokens x 32 planes: lanes have eight tokens each, eight of them and then the planes next to each other.
template <int DTYPE>
__global__ __launch_bounds__(256) void rotate_columns_kernel(RotateParams p, int interleaved) {
  typedef typename rotate_element<DTYPE>::type T;
  typedef Eight<DTYPE> Chunk;
  __shared__ RotationTile tile;
  tile.load(p, blockIdx.x * 64, blockIdx.y * kTilePlanes, kTilePlanes);
  const int token = blockIdx.x * 64 + threadIdx.x % 8 * 8, plane = blockIdx.y * kTilePlanes + threadIdx.x / 8;
  if (token >= p.tokens || plane >= p.dim / 2) return;
  const bool turned = plane < p.rotation.features / 2;
  const int count = min(8, p.tokens - token);
  int f0, f1;
  pair_of(p, plane, interleaved, f0, f1);
  float c[8], s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) c[i] = tile.c[threadIdx.x / 8][threadIdx.x % 8 * 8 + i], s[i] = tile.s[threadIdx.x / 8][threadIdx.x % 8 * 8 + i];
  const T* x = static_cast<const T*>(p.x) + token;
  T* out = static_cast<T*>(p.out) + token;
  const int first = blockIdx.z * p.per_thread, end = min(p.heads, first + p.per_thread);
  if (count < 8) {   // the last tokens
    for (int head = first; head < end; ++head)
#pragma unroll 1
      for (int i = 0; i < count; ++i) {
        const long long from = head * p.x_strides[1] + i, to = head * p.out_strides[1] + i;
        const T a = x[from + f0 * p.x_strides[2]], b = x[from + f1 * p.x_strides[2]];
        float y0 = widen<DTYPE>(a), y1 = widen<DTYPE>(b), ci = c[0], si = s[0];
#pragma unroll
        for (int j = 1; j < 8; ++j)
          if (i == j) ci = c[j], si = s[j];
        if (turned) rotate(y0, y1, ci, si);
        out[to + f0 * p.out_strides[2]] = turned ? narrow<DTYPE>(y0) : a, out[to + f1 * p.out_strides[2]] = turned ? narrow<DTYPE>(y1) : b;
      }
    return;
  }
  for (int head = first; head < end; head += kColumnsAhead) {
    Chunk a[kColumnsAhead], b[kColumnsAhead];
#pragma unroll
    for (int h = 0; h < kColumnsAhead; ++h) {
      if (head + h >= end) break;
      a[h].load(x + (head + h) * p.x_strides[1] + f0 * p.x_strides[2]);
      b[h].load(x + (head + h) * p.x_strides[1] + f1 * p.x_strides[2]);
    }
#pragma unroll
    for (int h = 0; h < kColumnsAhead; ++h) {
      if (head + h >= end) break;
      if (turned) {
        float y0[8], y1[8];
        a[h].get(y0), b[h].get(y1);
#pragma unroll
        for (int i = 0; i < 8; ++i) rotate(y0[i], y1[i], c[i], s[i]);
        a[h].set(y0), b[h].set(y1);
      }
      a[h].store(out + (head + h) * p.out_strides[1] + f0 * p.out_strides[2]);
      b[h].store(out + (head + h) * p.out_strides[1] + f1 * p.out_strides[2]);
    }
  }
}

// Workgroups of 64 tokens, a lane each, x up to 32 planes, in turn.  (16 bytes a lane at any alignment:
// 8191 tokens of 32 heads of 128 in fp16 66 us, 44 so.)
template <int DTYPE>
__global__ __launch_bounds__(256) void rotate_tokens_kernel(RotateParams p, int interleaved) {
  typedef typename rotate_element<DTYPE>::type T;
  __shared__ RotationTile tile;
  const int plane0 = blockIdx.y * p.planes, token = blockIdx.x * 64 + lane_id(), wave = uniform(threadIdx.x >> 6);
  tile.load(p, blockIdx.x * 64, plane0, p.planes);
  if (token >= p.tokens) return;
  const int first = blockIdx.z * p.per_thread, end = min(p.heads, first + p.per_thread), planes = min(p.dim / 2 - plane0, p.planes);
  const T* x = static_cast<const T*>(p.x) + token;
  T* out = static_cast<T*>(p.out) + token;
  for (int i = wave; i < planes; i += 4) {
    const bool turned = plane0 + i < p.rotation.features / 2;   // (uniform)
    int f0, f1;
    pair_of(p, plane0 + i, interleaved, f0, f1);
    const float c = tile.c[i][lane_id()], s = tile.s[i][lane_id()];
    for (int head = first; head < end; head += kColumnsAhead) {
      T a[kColumnsAhead], b[kColumnsAhead];
#pragma unroll
      for (int h = 0; h < kColumnsAhead; ++h) {
        if (head + h >= end) break;
        a[h] = x[(head + h) * p.x_strides[1] + f0 * p.x_strides[2]];
        b[h] = x[(head + h) * p.x_strides[1] + f1 * p.x_strides[2]];
      }
#pragma unroll
      for (int h = 0; h < kColumnsAhead; ++h) {
        if (head + h >= end) break;
        float y0 = widen<DTYPE>(a[h]), y1 = widen<DTYPE>(b[h]);
        if (turned) {
          rotate(y0, y1, c, s);
          a[h] = narrow<DTYPE>(y0), b[h] = narrow<DTYPE>(y1);
        }
        out[(head + h) * p.out_strides[1] + f0 * p.out_strides[2]] = a[h];
        out[(head + h) * p.out_strides[1] + f1 * p.out_strides[2]] = b[h];
      }
    }
  }
}

// Any strides, any even number of rotated features; a feature that has no partner is copied.
template <int DTYPE>
__global__ __launch_bounds__(256) void rotate_single_kernel(RotateParams p, int interleaved) {
  typedef typename rotate_element<DTYPE>::type T;
  const int planes = (p.dim + 1) / 2;
  const long long item = (long long)blockIdx.x * 256 + threadIdx.x;
  const int token = (int)(item / planes), plane = (int)(item % planes);
  if (token >= p.tokens) return;
  const bool turned = plane < p.rotation.features / 2;
  int f0, f1;
  pair_of(p, plane, interleaved, f0, f1);
  float c = 1.f, s = 0.f;
  if (turned) load_plane(p.rotation, token, plane, c, s);
  if (p.back) s = -s;
  const T* x = static_cast<const T*>(p.x) + token * p.x_strides[0];
  T* out = static_cast<T*>(p.out) + token * p.out_strides[0];
  for (int head = blockIdx.y; head < p.heads; head += gridDim.y) {
    const T a = x[head * p.x_strides[1] + f0 * p.x_strides[2]], b = f1 < p.dim ? x[head * p.x_strides[1] + f1 * p.x_strides[2]] : a;
    float y0 = widen<DTYPE>(a), y1 = widen<DTYPE>(b);
    if (turned) rotate(y0, y1, c, s);
    out[head * p.out_strides[1] + f0 * p.out_strides[2]] = turned ? narrow<DTYPE>(y0) : a;
    if (f1 < p.dim) out[head * p.out_strides[1] + f1 * p.out_strides[2]] = turned ? narrow<DTYPE>(y1) : b;
  }
}

const char* dtype_name(int dtype) { return dtype == IEX_F32 ? "f32" : dtype == IEX_BF16 ? "bf16" : "f16"; }

// Heads of a thread: all of them, fewer as long as the launch has too few workgroups.
int heads_of_a_thread(const RotateParams& p, long long workgroups, int ahead) {
  int per = p.heads;
  while (per > ahead && workgroups * ceil_div(p.heads, per) < 2048) per = (per / 2 + ahead - 1) / ahead * ahead;
  return per;
}

template <int DTYPE>
int launch(RotateParams p, bool interleaved, hipStream_t s) {
  constexpr int size = DTYPE == IEX_F32 ? 4 : 2, chunk = 16 / size;
  auto rows = [&](const void* x, const long long* strides) {
    return aligned(x, 16) && strides[2] == 1 && strides[0] % chunk == 0 && strides[1] % chunk == 0;
  };
  auto columns_aligned = [&](const void* x, const long long* strides) { return aligned(x, 16) && strides[1] % chunk == 0 && strides[2] % chunk == 0; };
  if (p.dim % 16 == 0 && p.rotation.features % 16 == 0 && rows(p.x, p.x_strides) && rows(p.out, p.out_strides)) {
    const long long grid = ceil_div((long long)p.tokens * (p.dim / 16), 256);
    p.per_thread = heads_of_a_thread(p, grid, kRowsAhead);
    const dim3 dims((unsigned)grid, ceil_div(p.heads, p.per_thread));
    note_kernel("rotate_rows_kernel<%s>", dtype_name(DTYPE));
    if (interleaved) hipLaunchKernelGGL((rotate_rows_kernel<DTYPE, true>), dims, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((rotate_rows_kernel<DTYPE, false>), dims, dim3(256), 0, s, p);
  } else if (p.dim % 2 == 0 && p.x_strides[0] == 1 && p.out_strides[0] == 1 && p.tokens >= 8) {
    const bool whole = columns_aligned(p.x, p.x_strides) && columns_aligned(p.out, p.out_strides);
    auto grid = [&] { return (long long)ceil_div(p.tokens, 64) * ceil_div(p.dim, 2 * p.planes); };
    p.planes = kTilePlanes;
    // (a wavefront's planes come one after the other: fewer of them where there are too few workgroups; 2001 tokens of 8 heads 17.3 us by 32)
    while (!whole && p.planes > 4 && grid() * ceil_div(p.heads, kColumnsAhead) < 1024) p.planes /= 2;
    p.per_thread = heads_of_a_thread(p, grid(), kColumnsAhead);
    const dim3 dims(ceil_div(p.tokens, 64), ceil_div(p.dim, 2 * p.planes), ceil_div(p.heads, p.per_thread));
    note_kernel("%s<%s>", whole ? "rotate_columns_kernel" : "rotate_tokens_kernel", dtype_name(DTYPE));
    if (whole) hipLaunchKernelGGL((rotate_columns_kernel<DTYPE>), dims, dim3(256), 0, s, p, interleaved);
    else hipLaunchKernelGGL((rotate_tokens_kernel<DTYPE>), dims, dim3(256), 0, s, p, interleaved);
  } else {
    const long long grid = ceil_div((long long)p.tokens * ((p.dim + 1) / 2), 256);
    note_kernel("rotate_single_kernel<%s>", dtype_name(DTYPE));
    hipLaunchKernelGGL((rotate_single_kernel<DTYPE>), dim3((unsigned)grid, grid >= 2048 ? ceil_div(p.heads, 4) : p.heads), dim3(256), 0, s, p, interleaved);
  }
  return check_hip(hipGetLastError(), "rotate launch");
}

}  // namespace
}  // namespace iex

extern "C" int iex_rotate(int dtype, int tokens, int heads, int head_dim, const void* x, const long long* x_strides, void* out, const long long* out_strides,
                          const iex_rotation* rotation, int back, void* stream) {
  using namespace iex;
  trail_reset();
  IEX_REQUIRE(dtype == IEX_F32 || dtype == IEX_F16 || dtype == IEX_BF16, IEX_ERR_UNSUPPORTED, "rotate: fp32, fp16 or bf16");
  IEX_REQUIRE(tokens >= 0 && heads >= 0 && head_dim >= 0, IEX_ERR_BAD_ARGUMENT, "rotate: negative dimension");
  if (tokens == 0) return 0;
  IEX_REQUIRE(rotation && rotation->at, IEX_ERR_BAD_ARGUMENT, "rotate: null pointer argument");
  RotateParams p{};
  if (int rc = check_rotation(rotation, "rotate", p.rotation)) return rc;
  IEX_REQUIRE(p.rotation.features % 2 == 0 && p.rotation.features <= head_dim, IEX_ERR_UNSUPPORTED, "rotate: rotated features must be an even number of the head's (%d of %d)",
              p.rotation.features, head_dim);
  if (heads == 0 || head_dim == 0) return 0;
  IEX_REQUIRE(x && out && x_strides && out_strides, IEX_ERR_BAD_ARGUMENT, "rotate: null pointer argument");
  IEX_REQUIRE(aligned(x, dtype == IEX_F32 ? 4 : 2) && aligned(out, dtype == IEX_F32 ? 4 : 2), IEX_ERR_UNSUPPORTED, "rotate: operands must be aligned to their elements");
  IEX_REQUIRE((long long)tokens * ((head_dim + 1) / 2) < (1ll << 31) && heads < 65536 && head_dim < 65536, IEX_ERR_TOO_LARGE, "rotate: too many tokens or heads");
  p.tokens = tokens, p.heads = heads, p.dim = head_dim, p.back = back, p.x = x, p.out = out;
  for (int i = 0; i < 3; ++i) p.x_strides[i] = x_strides[i], p.out_strides[i] = out_strides[i];
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == IEX_F32) return launch<IEX_F32>(p, rotation->interleaved, s);
  return dtype == IEX_BF16 ? launch<IEX_BF16>(p, rotation->interleaved, s) : launch<IEX_F16>(p, rotation->interleaved, s);
}
