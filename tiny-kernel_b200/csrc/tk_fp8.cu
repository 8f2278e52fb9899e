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
// the groups' maxima and the codes.  A thread has 32 bytes of consecutive values of a group, so 16 lanes share it, of
// 16-bit types 8.  us, and the bytes at the rate of a copy: norm 8192 x 4096 bf16 45.8, 36.5; rows 2048 x 14336 bf16
// 15.4, 13.8; weight 14336 x 4096 f32 45.9, 45.5; norm 4 x 4096 f32 2.6, which is a launch's way through the SMs.  Rows that
// are not whole chunks, or off their boundary, go by elements, 8 or 16 neighbours a thread, which is several times as
// long: 8192 x 2000 and 2008 bf16 26 and 145, as rows alone 9.7 and 47.  f32 rows wider than 8192 have four chunks a
// thread in 64 registers and spill some: 2048 x 8192 and 16384 f32 43 and 94, for 34 and 68.
#include <algorithm>
#include <cstring>
#include <type_traits>

#include "tk_elements.cuh"
#include "tk_fp8.h"
#include "tk_kv4.h"

namespace tk {
namespace {

template <class T>
constexpr int kChunk = 32 / sizeof(T);  // values of a thread's chunk
constexpr float kLargest = 448.f, kLeastScale = 1.17549435e-38f;  // of e4m3; 2^-126

// Whether every row of values lies on a boundary of 16 bytes.
template <class T>
bool even(const void* base, long long stride) {
  return (reinterpret_cast<uintptr_t>(base) | (uintptr_t)(stride * (long long)sizeof(T))) % 16 == 0;
}

// A thread's chunk as it lies in memory.  FAST: rows on 16-byte boundaries and of whole chunks, so that loads are of 16
// bytes; all of a thread's are on their way before the first is looked at (loads that were converted one after the
// other took bf16 rows longer than f32 ones).  Otherwise by elements.
template <class T, int E, bool FAST>
struct Chunk {
  static constexpr int kLoads = FAST ? (int)sizeof(T) * E / 16 : 1;
  uint4 raw[kLoads];
  T e[FAST ? 1 : E];
  __device__ __forceinline__ void load(const T* src, int n) {
    if constexpr (FAST) {
#pragma unroll
      for (int w = 0; w < kLoads; ++w) raw[w] = n <= 0 ? make_uint4(0, 0, 0, 0) : reinterpret_cast<const uint4*>(src)[w];
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) e[i] = i < n ? src[i] : from_f32<T>(0.f);
    }
  }
  __device__ __forceinline__ void values(float (&v)[E]) const {
    if constexpr (!FAST) {
#pragma unroll
      for (int i = 0; i < E; ++i) v[i] = to_f32(e[i]);
    } else {
#pragma unroll
      for (int l = 0; l < kLoads; ++l) {
        const uint32_t w[4] = {raw[l].x, raw[l].y, raw[l].z, raw[l].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (sizeof(T) == 4) {
            v[4 * l + i] = __uint_as_float(w[i]);
          } else if constexpr (std::is_same<T, __half>::value) {
            const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            v[8 * l + 2 * i] = y.x, v[8 * l + 2 * i + 1] = y.y;
          } else {
            v[8 * l + 2 * i] = __uint_as_float(w[i] << 16), v[8 * l + 2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
          }
        }
      }
    }
  }
};
template <class T, int E, bool FAST>
__device__ __forceinline__ void store_chunk(T* dst, int n, const float (&v)[E]) {
  if constexpr (FAST) {
    store_f32<T, E>(dst, 1, v);
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (i < n) dst[i] = from_f32<T>(v[i]);
  }
}

// Largest magnitude as bits: those of infinities and NaNs are above all others'.
template <int E>
__device__ __forceinline__ uint32_t largest_bits(const float (&v)[E]) {
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < E; ++i) most = max(most, __float_as_uint(v[i]) & 0x7fffffffu);
  return most;
}
// The same of a chunk as it lies in memory: of 16-bit types two at once, whose magnitudes are in the order of their bits.
template <class T, int E, bool FAST>
__device__ __forceinline__ uint32_t largest_bits(const Chunk<T, E, FAST>& x, const float (&v)[E]) {
  if constexpr (FAST && sizeof(T) == 2) {
    uint32_t most = 0;
#pragma unroll
    for (int l = 0; l < Chunk<T, E, FAST>::kLoads; ++l) {
      most = __vmaxu2(most, x.raw[l].x & 0x7fff7fffu);
      most = __vmaxu2(most, x.raw[l].y & 0x7fff7fffu);
      most = __vmaxu2(most, x.raw[l].z & 0x7fff7fffu);
      most = __vmaxu2(most, x.raw[l].w & 0x7fff7fffu);
    }
    const uint16_t bits = (uint16_t)max(most & 0xffffu, most >> 16);
    T y;
    memcpy(&y, &bits, 2);
    return __float_as_uint(to_f32(y));
  } else {
    return largest_bits(v);
  }
}
// Of the lanes that share a group.
template <int LANES>
__device__ __forceinline__ uint32_t of_group(uint32_t most) {
#pragma unroll
  for (int off = LANES / 2; off; off >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, off));
  return most;
}

struct GroupScale {
  float scale, over;  // and 1 / scale; 0 of a group that is not finite
};
__device__ __forceinline__ GroupScale group_scale(uint32_t most) {
  if (most >= 0x7f800000u) return {__uint_as_float(0x7fc00000u), 0.f};
  const float s = fmaxf(__fdiv_rn(__uint_as_float(most), kLargest), kLeastScale);
  return {s, __frcp_rn(s)};
}

// Codes of v[0] / scale .. v[3] / scale.  A product with the reciprocal alone would round some quotients to the wrong
// side of a tie, of which 16-bit values over their largest make many (7 codes in 10000, bf16); it is corrected by its
// remainder, after which it is the nearest f32 (Markstein, 1990), unless the remainder is below the least f32: values
// below about 1e-30.  (With divisions 22 us instead of 15: 2048 x 14336 bf16.)
__device__ __forceinline__ uint32_t codes4(const float* v, const GroupScale& g) {
  const unsigned long long over = pair_of(g.over, g.over), less = pair_of(-g.scale, -g.scale);
  uint32_t y = 0;
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    const unsigned long long x = pair_of(v[i], v[i + 1]), q = mul2(x, over);
    const float2 r = values_of(fma2(fma2(q, less, x), over, q));
    uint16_t two;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(two) : "f"(r.y), "f"(r.x));
    y |= (uint32_t)two << (8 * i);
  }
  return y;
}
// FAST: dst is on a boundary of E bytes.
template <int E, bool FAST>
__device__ __forceinline__ void store_codes(uint8_t* dst, int n, const float (&v)[E], const GroupScale& g) {
  uint32_t y[E / 4];
#pragma unroll
  for (int i = 0; i < E / 4; ++i) {
    y[i] = codes4(&v[4 * i], g);
    if (g.over == 0.f) y[i] = 0;
  }
  if constexpr (!FAST) {
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (i < n) dst[i] = (uint8_t)(y[i / 4] >> (i % 4 * 8));
  } else if constexpr (E == 8) {
    *reinterpret_cast<uint2*>(dst) = make_uint2(y[0], y[1]);
  } else {
    *reinterpret_cast<uint4*>(dst) = make_uint4(y[0], y[1], y[2], y[3]);
  }
}

// ---- norm ------------------------------------------------------------------------------------------

// `warps` warps a row, V chunks a thread; a block has as many rows as its warps make.
template <class T, int V, int THREADS, bool FAST>
__global__ void __launch_bounds__(THREADS) add_rmsnorm_fp8_kernel(Fp8RowsParams p, int warps) {
  constexpr int kE = kChunk<T>, kLanes = kFp8Block / kE;
  __shared__ float part[32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, first = warp / warps * warps;
  const long long row = (long long)blockIdx.x * (blockDim.x / 32 / warps) + warp / warps;
  const bool live = row < p.rows;
  const int at = ((warp - first) * 32 + lane) * kE, step = warps * 32 * kE;
  after_previous();
  Chunk<T, kE, FAST> x[V], r[V];
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
    if (p.sum && n > 0) store_chunk<T, kE, FAST>(static_cast<T*>(p.sum) + row * p.sum_stride + e, n, v[i]);
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
      Chunk<float, kE, FAST> w;
      float y[kE];
      w.load(p.weight + e, n);
      w.values(y);
#pragma unroll
      for (int j = 0; j < kE; ++j) v[i][j] = v[i][j] * rms * y[j];
    } else {
#pragma unroll
      for (int j = 0; j < kE; ++j) v[i][j] *= rms;
    }
    const GroupScale g = group_scale(of_group<kLanes>(largest_bits(v[i])));
    if (n > 0) {
      store_codes<kE, FAST>(p.codes + row * p.codes_stride + e, n, v[i], g);
      if (lane % kLanes == 0) p.scales[row * ((p.dim + kFp8Block - 1) / kFp8Block) + e / kFp8Block] = g.scale;
    }
  }
}

template <class T, int V, int THREADS>
cudaError_t launch_norm(const Fp8RowsParams& p, bool fast, int warps, int block_rows, cudaStream_t st) {
  const dim3 blocks(((unsigned)p.rows + block_rows - 1) / block_rows);
  const int threads = block_rows * warps * 32;
  if (fast) return launch(add_rmsnorm_fp8_kernel<T, V, THREADS, true>, blocks, threads, 0, st, p, warps);
  return launch(add_rmsnorm_fp8_kernel<T, V, THREADS, false>, blocks, threads, 0, st, p, warps);
}

template <class T>
bool even_codes(const Fp8RowsParams& p) {
  return p.dim % kChunk<T> == 0 && (reinterpret_cast<uintptr_t>(p.codes) | (uintptr_t)p.codes_stride) % kChunk<T> == 0;
}

template <class T>
cudaError_t launch_norm(const Fp8RowsParams& p, int sm_count, cudaStream_t st) {
  const bool fast = even<T>(p.x, p.x_stride) && (!p.residual || even<T>(p.residual, p.residual_stride)) &&
                    (!p.sum || even<T>(p.sum, p.sum_stride)) && even<float>(p.weight, 0) && even_codes<T>(p);
  const int chunks = (p.dim + kChunk<T> - 1) / kChunk<T>;
  // Few rows: as many threads as a row has chunks.  Many: 128 bytes of f32, 64 of 16-bit types a thread.
  constexpr int kMost = sizeof(T) == 4 ? 4 : 2;
  int v = p.rows < 2 * sm_count ? 1 : kMost;
  while (v > 1 && chunks <= 32 * (v / 2)) v /= 2;
  while ((chunks + v * 32 - 1) / (v * 32) > 32) v *= 2;
  const int warps = (chunks + v * 32 - 1) / (v * 32);
  const int block_rows = p.rows < 2 * sm_count ? 1 : std::max(1, 4 / warps);
  if (v == 1) return launch_norm<T, 1, 1024>(p, fast, warps, block_rows, st);
  if (v == kMost && warps <= 8) return launch_norm<T, kMost, 256>(p, fast, warps, block_rows, st);
  if (v == 2) return launch_norm<T, 2, 1024>(p, fast, warps, block_rows, st);
  return launch_norm<T, kMost, 1024>(p, fast, warps, block_rows, st);
}

// ---- rows and blocks as they are -----------------------------------------------------------------------

constexpr int kThreads = 256;

template <class T, bool FAST>
__global__ void __launch_bounds__(kThreads) fp8_quantize_rows_kernel(Fp8RowsParams p, unsigned groups, unsigned total) {
  constexpr int kE = kChunk<T>, kLanes = kFp8Block / kE;
  after_previous();
  // (a thread with two or four groups was slower by 3 and 15 %: 2048 x 14336 bf16)
  const unsigned group = blockIdx.x * (kThreads / kLanes) + threadIdx.x / kLanes;  // (threads may be more than 2^32)
  const int lane = threadIdx.x % kLanes, at = (int)(group % groups) * kFp8Block + lane * kE;
  const long long row = group / groups;
  const int n = group < total ? p.dim - at : 0;
  Chunk<T, kE, FAST> x;
  x.load(static_cast<const T*>(p.x) + row * p.x_stride + at, n);
  float v[kE];
  x.values(v);
  const GroupScale g = group_scale(of_group<kLanes>(largest_bits(x, v)));
  if (n <= 0) return;
  store_codes<kE, FAST>(p.codes + row * p.codes_stride + at, n, v, g);
  if (lane == 0) p.scales[group] = g.scale;
}

template <class T, bool FAST>
__global__ void __launch_bounds__(kThreads) fp8_quantize_blocks_kernel(Fp8RowsParams p, unsigned groups) {
  constexpr int kE = kChunk<T>, kLanes = kFp8Block / kE, kRows = kThreads / kLanes, kTurns = kFp8Block / kRows;
  __shared__ uint32_t part[kThreads / 32];
  after_previous();
  const long long block = blockIdx.x / groups;
  const int at = (int)(blockIdx.x % groups) * kFp8Block + threadIdx.x % kLanes * kE;
  Chunk<T, kE, FAST> x[kTurns];
  uint32_t most = 0;
  const long long row0 = block * kFp8Block + threadIdx.x / kLanes;
#pragma unroll
  for (int t = 0; t < kTurns; ++t) {
    const long long row = row0 + t * kRows;
    x[t].load(static_cast<const T*>(p.x) + row * p.x_stride + at, row < p.rows ? p.dim - at : 0);
  }
  float v[kE];
#pragma unroll
  for (int t = 0; t < kTurns; ++t) {
    x[t].values(v);
    most = max(most, largest_bits(x[t], v));
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
    if (row < p.rows && at < p.dim) {
      x[t].values(v);
      store_codes<kE, FAST>(p.codes + row * p.codes_stride + at, p.dim - at, v, g);
    }
  }
  if (threadIdx.x == 0) p.scales[blockIdx.x] = g.scale;
}

template <class T>
cudaError_t launch_quantize(const Fp8RowsParams& p, int block_rows, cudaStream_t st) {
  const bool fast = even<T>(p.x, p.x_stride) && even_codes<T>(p);
  const unsigned groups = (unsigned)((p.dim + kFp8Block - 1) / kFp8Block);
  if (block_rows == 1) {
    const unsigned total = groups * (unsigned)p.rows;
    constexpr unsigned kEach = kThreads * kChunk<T> / kFp8Block;
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
