// tk_fp8.cu -- what becomes the operands of the 8-bit product: rows with a scale for each group of 128, with or
// without the residual's addition and the RMS norm before, and weights in blocks of 128 x 128.
//
//   s = x + residual,  y = s * rsqrt(mean(s^2) + eps) * weight        (without the norm: y = x)
//   a = max |y| of the group,  scale = max(a / 448, 2^-126),  code = e4m3(y / scale), to the nearest
//
// s is kept in f32 and only its copy for the residual stream is rounded, so the norm does not see that rounding.
// The least scale keeps a group of zeros, or of subnormals, from dividing by nothing.  A group that holds an
// infinity or a NaN gets the scale NaN: it reads back as NaN, and so does every sum over it.
//
// Bound by memory: one pass, every value is read once into registers and stays there between the sum of squares,
// the groups' maxima and the codes.  A thread has eight consecutive values of a group, so 16 lanes share it.
#include <algorithm>
#include <type_traits>

#include "tk_elements.cuh"
#include "tk_fp8.h"
#include "tk_kv4.h"

namespace tk {
namespace {

constexpr int kE = 8;  // values of a thread's chunk: 16 bytes of 16-bit types, 8 bytes of codes
constexpr float kLargest = 448.f, kLeastScale = 1.17549435e-38f;  // of e4m3; 2^-126

// Whether every row of values lies on a boundary of 16 bytes.
template <class T>
bool even(const void* base, long long stride) {
  return (reinterpret_cast<uintptr_t>(base) | (uintptr_t)(stride * (long long)sizeof(T))) % 16 == 0;
}

// A thread's chunk as it lies in memory.  FAST: rows on 16-byte boundaries and of whole chunks, so that a load is 16 or 32
// bytes; all of a thread's are on their way before the first is looked at (loads that were converted one after the
// other took bf16 rows longer than f32 ones).  Otherwise by elements.
template <class T, bool FAST>
struct Chunk {
  uint4 raw[FAST ? sizeof(T) * kE / 16 : 1];
  T e[FAST ? 1 : kE];
  __device__ __forceinline__ void load(const T* src, int n) {
    if constexpr (FAST) {
      if (n <= 0) {
#pragma unroll
        for (int w = 0; w < (int)sizeof(T) * kE / 16; ++w) raw[w] = make_uint4(0, 0, 0, 0);
      } else if constexpr (sizeof(T) == 4) {
        raw[0] = reinterpret_cast<const uint4*>(src)[0];
        raw[1] = reinterpret_cast<const uint4*>(src)[1];
      } else {
        raw[0] = *reinterpret_cast<const uint4*>(src);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kE; ++i) e[i] = i < n ? src[i] : from_f32<T>(0.f);
    }
  }
  __device__ __forceinline__ void values(float (&v)[kE]) const {
    if constexpr (!FAST) {
#pragma unroll
      for (int i = 0; i < kE; ++i) v[i] = to_f32(e[i]);
    } else if constexpr (sizeof(T) == 4) {
      const uint32_t w[8] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w, raw[1].x, raw[1].y, raw[1].z, raw[1].w};
#pragma unroll
      for (int i = 0; i < kE; ++i) v[i] = __uint_as_float(w[i]);
    } else {
      const uint32_t w[4] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same<T, __half>::value) {
          const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
          v[2 * i] = y.x, v[2 * i + 1] = y.y;
        } else {
          v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
      }
    }
  }
};
template <class T, bool FAST>
__device__ __forceinline__ void store_chunk(T* dst, int n, const float (&v)[kE]) {
  if constexpr (FAST) {
    store_f32<T, kE>(dst, 1, v);
  } else {
#pragma unroll
    for (int i = 0; i < kE; ++i)
      if (i < n) dst[i] = from_f32<T>(v[i]);
  }
}

// Largest magnitude as bits: those of infinities and NaNs are above all others'.
__device__ __forceinline__ uint32_t largest_bits(const float (&v)[kE]) {
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < kE; ++i) most = max(most, __float_as_uint(v[i]) & 0x7fffffffu);
  return most;
}

struct GroupScale {
  float scale, over;  // and 1 / scale; 0 of a group that is not finite
};
__device__ __forceinline__ GroupScale group_scale(uint32_t most) {
  if (most >= 0x7f800000u) return {__uint_as_float(0x7fc00000u), 0.f};
  const float s = fmaxf(__uint_as_float(most) / kLargest, kLeastScale);
  return {s, 1.f / s};
}

__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return lo | (uint32_t)hi << 16;
}
// FAST: dst is on an 8-byte boundary.
template <bool FAST>
__device__ __forceinline__ void store_codes(uint8_t* dst, int n, const float (&v)[kE], const GroupScale& g) {
  uint2 y = make_uint2(0, 0);
  if (g.over != 0.f) {
    y.x = codes4(v[0] * g.over, v[1] * g.over, v[2] * g.over, v[3] * g.over);
    y.y = codes4(v[4] * g.over, v[5] * g.over, v[6] * g.over, v[7] * g.over);
  }
  if (FAST) {
    *reinterpret_cast<uint2*>(dst) = y;
  } else {
#pragma unroll
    for (int i = 0; i < kE; ++i)
      if (i < n) dst[i] = (uint8_t)((i < 4 ? y.x : y.y) >> (i % 4 * 8));
  }
}

// ---- norm ------------------------------------------------------------------------------------------

// `warps` warps a row, V chunks a thread; a block has as many rows as its warps make.
template <class T, int V, int THREADS, bool FAST>
__global__ void __launch_bounds__(THREADS) add_rmsnorm_fp8_kernel(Fp8RowsParams p, int warps) {
  __shared__ float part[32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, first = warp / warps * warps;
  const long long row = (long long)blockIdx.x * (blockDim.x / 32 / warps) + warp / warps;
  const bool live = row < p.rows;
  const int at = ((warp - first) * 32 + lane) * kE, step = warps * 32 * kE;
  after_previous();
  Chunk<T, FAST> x[V], r[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = at + i * step, n = live ? p.dim - e : 0;
    x[i].load(static_cast<const T*>(p.x) + row * p.x_stride + e, n);
    if (p.residual) r[i].load(static_cast<const T*>(p.residual) + row * p.residual_stride + e, n);
  }
  float v[V][kE];
  float squares = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = at + i * step, n = live ? p.dim - e : 0;
    x[i].values(v[i]);
    if (p.residual) {
      float y[kE];
      r[i].values(y);
#pragma unroll
      for (int j = 0; j < kE; ++j) v[i][j] += y[j];
    }
    if (p.sum && n > 0) store_chunk<T, FAST>(static_cast<T*>(p.sum) + row * p.sum_stride + e, n, v[i]);
#pragma unroll
    for (int j = 0; j < kE; ++j) squares = fmaf(v[i][j], v[i][j], squares);
  }
#pragma unroll
  for (int off = 16; off; off >>= 1) squares += __shfl_xor_sync(0xffffffffu, squares, off);
  if (warps > 1) {
    if (lane == 0) part[warp] = squares;
    __syncthreads();
    squares = 0.f;
    for (int w = 0; w < warps; ++w) squares += part[first + w];
  }
  const float rms = rsqrtf(squares / (float)p.dim + p.eps);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = at + i * step, n = live ? p.dim - e : 0;
    if (p.weight) {
      Chunk<float, FAST> w;
      float y[kE];
      w.load(p.weight + e, n);
      w.values(y);
#pragma unroll
      for (int j = 0; j < kE; ++j) v[i][j] = v[i][j] * rms * y[j];
    } else {
#pragma unroll
      for (int j = 0; j < kE; ++j) v[i][j] *= rms;
    }
    uint32_t most = largest_bits(v[i]);
#pragma unroll
    for (int off = 8; off; off >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, off));
    const GroupScale g = group_scale(most);
    if (n > 0) {
      store_codes<FAST>(p.codes + row * p.codes_stride + e, n, v[i], g);
      if (lane % 16 == 0) p.scales[row * ((p.dim + kFp8Block - 1) / kFp8Block) + e / kFp8Block] = g.scale;
    }
  }
}

template <class T, int V, int THREADS>
cudaError_t launch_norm(const Fp8RowsParams& p, bool fast, int warps, int block_rows, cudaStream_t st) {
  const dim3 blocks((unsigned)((p.rows + block_rows - 1) / block_rows));
  const int threads = block_rows * warps * 32;
  if (fast) return launch(add_rmsnorm_fp8_kernel<T, V, THREADS, true>, blocks, threads, 0, st, p, warps);
  return launch(add_rmsnorm_fp8_kernel<T, V, THREADS, false>, blocks, threads, 0, st, p, warps);
}

bool even_codes(const Fp8RowsParams& p) {
  return p.dim % kE == 0 && (reinterpret_cast<uintptr_t>(p.codes) | (uintptr_t)p.codes_stride) % 8 == 0;
}

template <class T>
cudaError_t launch_norm(const Fp8RowsParams& p, int sm_count, cudaStream_t st) {
  const bool fast = even<T>(p.x, p.x_stride) && (!p.residual || even<T>(p.residual, p.residual_stride)) &&
                    (!p.sum || even<T>(p.sum, p.sum_stride)) && even<float>(p.weight, 0) && even_codes(p);
  const int chunks = (p.dim + kE - 1) / kE;
  // Few rows: as many threads as a row has chunks.  Many: four chunks a thread.
  int v = p.rows < 2 * sm_count ? 1 : 4;
  while (v > 1 && chunks <= 32 * (v / 2)) v /= 2;
  while ((chunks + v * 32 - 1) / (v * 32) > 32) v *= 2;
  const int warps = (chunks + v * 32 - 1) / (v * 32);
  const int block_rows = p.rows < 2 * sm_count ? 1 : std::max(1, 4 / warps);
  if (v == 1) return launch_norm<T, 1, 1024>(p, fast, warps, block_rows, st);
  if (v == 2) return launch_norm<T, 2, 1024>(p, fast, warps, block_rows, st);
  if (warps > 8) return launch_norm<T, 4, 1024>(p, fast, warps, block_rows, st);
  return launch_norm<T, 4, 256>(p, fast, warps, block_rows, st);
}

// ---- rows and blocks as they are -----------------------------------------------------------------------

constexpr int kThreads = 256;
constexpr int kUnroll = 4;  // groups of a half warp, all loaded before the first is used

template <class T, bool FAST>
__global__ void __launch_bounds__(kThreads) fp8_quantize_rows_kernel(Fp8RowsParams p, unsigned groups, unsigned total) {
  after_previous();
  const unsigned half = (blockIdx.x * kThreads + threadIdx.x) / 16;
  const int lane = threadIdx.x % 16;
  Chunk<T, FAST> x[kUnroll];
  long long row[kUnroll];
  int at[kUnroll], n[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const unsigned g = half + u * gridDim.x * (kThreads / 16);
    row[u] = g / groups;
    at[u] = (int)(g % groups) * kFp8Block + lane * kE;
    n[u] = g < total ? p.dim - at[u] : 0;
    x[u].load(static_cast<const T*>(p.x) + row[u] * p.x_stride + at[u], n[u]);
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    float v[kE];
    x[u].values(v);
    uint32_t most = largest_bits(v);
#pragma unroll
    for (int off = 8; off; off >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, off));
    const GroupScale g = group_scale(most);
    if (n[u] > 0) {
      store_codes<FAST>(p.codes + row[u] * p.codes_stride + at[u], n[u], v, g);
      if (lane == 0) p.scales[row[u] * groups + at[u] / kFp8Block] = g.scale;
    }
  }
}

template <class T, bool FAST>
__global__ void __launch_bounds__(kThreads) fp8_quantize_blocks_kernel(Fp8RowsParams p, unsigned groups) {
  __shared__ uint32_t part[kThreads / 32];
  after_previous();
  constexpr int kRows = kThreads / 16, kTurns = kFp8Block / kRows;
  const long long block = blockIdx.x / groups;
  const int at = (int)(blockIdx.x % groups) * kFp8Block + threadIdx.x % 16 * kE;
  Chunk<T, FAST> x[kTurns];
  uint32_t most = 0;
  const long long row0 = block * kFp8Block + threadIdx.x / 16;
#pragma unroll
  for (int t = 0; t < kTurns; ++t) {
    const long long row = row0 + t * kRows;
    x[t].load(static_cast<const T*>(p.x) + row * p.x_stride + at, row < p.rows ? p.dim - at : 0);
  }
  float v[kTurns][kE];
#pragma unroll
  for (int t = 0; t < kTurns; ++t) {
    x[t].values(v[t]);
    most = max(most, largest_bits(v[t]));
  }
  most = __reduce_max_sync(0xffffffffu, most);
  if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) most = max(most, part[w]);
  const GroupScale g = group_scale(most);
#pragma unroll
  for (int t = 0; t < kTurns; ++t) {
    const long long row = row0 + t * kRows;
    if (row < p.rows && at < p.dim) store_codes<FAST>(p.codes + row * p.codes_stride + at, p.dim - at, v[t], g);
  }
  if (threadIdx.x == 0) p.scales[blockIdx.x] = g.scale;
}

template <class T>
cudaError_t launch_quantize(const Fp8RowsParams& p, int block_rows, cudaStream_t st) {
  const bool fast = even<T>(p.x, p.x_stride) && even_codes(p);
  const unsigned groups = (unsigned)((p.dim + kFp8Block - 1) / kFp8Block);
  if (block_rows == 1) {
    const unsigned total = groups * (unsigned)p.rows;
    constexpr unsigned kEach = kThreads / 16 * kUnroll;
    const dim3 blocks((total + kEach - 1) / kEach);
    if (fast) return launch(fp8_quantize_rows_kernel<T, true>, blocks, kThreads, 0, st, p, groups, total);
    return launch(fp8_quantize_rows_kernel<T, false>, blocks, kThreads, 0, st, p, groups, total);
  }
  const dim3 blocks(groups * (unsigned)(((long long)p.rows + kFp8Block - 1) / kFp8Block));
  if (fast) return launch(fp8_quantize_blocks_kernel<T, true>, blocks, kThreads, 0, st, p, groups);
  return launch(fp8_quantize_blocks_kernel<T, false>, blocks, kThreads, 0, st, p, groups);
}

}  // namespace

cudaError_t launch_add_rmsnorm_fp8(const Fp8RowsParams& p, int dtype, int sm_count, cudaStream_t st) {
  if (dtype == kTypeF32) return launch_norm<float>(p, sm_count, st);
  return dtype == kTypeBF16 ? launch_norm<__nv_bfloat16>(p, sm_count, st) : launch_norm<__half>(p, sm_count, st);
}

cudaError_t launch_fp8_quantize(const Fp8RowsParams& p, int block_rows, int dtype, cudaStream_t st) {
  if (dtype == kTypeF32) return launch_quantize<float>(p, block_rows, st);
  return dtype == kTypeBF16 ? launch_quantize<__nv_bfloat16>(p, block_rows, st)
                            : launch_quantize<__half>(p, block_rows, st);
}

}  // namespace tk
