// tk_elements.cuh -- what the kernels of the serving step share: programmatic launches, elements of each
// type as f32.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace tk {
namespace {

// Programmatic launches: a kernel is set up while the one before it in the stream runs; it reads
// nothing, and no thread of it ends, before that one has completed.  It reads nothing through the
// read-only path (__ldg) either, which holds only for what no kernel writes once it has been set up.
__device__ __forceinline__ void after_previous() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
template <class... P, class... A>
cudaError_t launch(void (*kernel)(P...), dim3 blocks, int threads, size_t smem, cudaStream_t st, A... args) {
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = blocks;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

// ---- elements ------------------------------------------------------------------------------------

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// E consecutive elements as f32.  vec: the address is on a 16-byte boundary (E elements are 16 or
// 32 bytes), 2: on a 32-byte boundary.
template <class T, int E>
__device__ __forceinline__ void load_f32(const T* src, int vec, float (&v)[E]) {
  if constexpr (E * sizeof(T) == 32) {
    if (vec == 2) {
      static_assert(sizeof(T) == 4, "");
      asm volatile("ld.global.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                   : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
                   : "l"(src));
      return;
    }
  }
  if (vec) {
    constexpr int W = E * (int)sizeof(T) / 16;
    uint4 raw[W];
#pragma unroll
    for (int w = 0; w < W; ++w) raw[w] = reinterpret_cast<const uint4*>(src)[w];
    const T* e = reinterpret_cast<const T*>(raw);
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = to_f32(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = to_f32(src[i]);
  }
}

// Rounds once, to the nearest of T.
template <class T, int E>
__device__ __forceinline__ void store_f32(T* dst, int vec, const float (&v)[E]) {
  if constexpr (E * sizeof(T) == 32) {
    if (vec == 2) {
      asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(dst), "f"(v[0]), "f"(v[1]), "f"(v[2]),
                   "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
                   : "memory");
      return;
    }
  }
  if (vec) {
    constexpr int W = E * (int)sizeof(T) / 16;
    uint4 raw[W];
    T* e = reinterpret_cast<T*>(raw);
#pragma unroll
    for (int i = 0; i < E; ++i) e[i] = from_f32<T>(v[i]);
#pragma unroll
    for (int w = 0; w < W; ++w) reinterpret_cast<uint4*>(dst)[w] = raw[w];
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) dst[i] = from_f32<T>(v[i]);
  }
}

// Two f32 at once.
__device__ __forceinline__ unsigned long long pair_of(float a, float b) {
  unsigned long long y;
  asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float2 values_of(unsigned long long p) {
  float2 y;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(y.x), "=f"(y.y) : "l"(p));
  return y;
}
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
  unsigned long long y;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(y) : "l"(a), "l"(b), "l"(c));
  return y;
}
__device__ __forceinline__ unsigned long long mul2(unsigned long long a, unsigned long long b) {
  unsigned long long y;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(a), "l"(b));
  return y;
}

}  // namespace
}  // namespace tk
