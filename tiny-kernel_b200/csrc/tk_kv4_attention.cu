// tk_kv4_attention.cu -- attention over the key/value cache held in 4 bits.
//
// For query i of the n query tokens of a sequence with kv_len tokens in the cache (those n among
// them): o = sum_p w_p v_p, w = softmax_p(scale * q . k_p) over the positions p < kv_len - n + i + 1,
// with k, v = code * scale + offset.  A position whose page is not in the cache counts as absent; a
// query that sees no position gets zeros.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "tk_kv4.h"

namespace tk {
namespace {

__device__ __forceinline__ float load_any(const void* base, long long i, int dtype) {
  if (dtype == kTypeF32) return static_cast<const float*>(base)[i];
  if (dtype == kTypeF16) return __half2float(static_cast<const __half*>(base)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(base)[i]);
}
__device__ __forceinline__ void store_any(void* base, long long i, int dtype, float v) {
  if (dtype == kTypeF32)
    static_cast<float*>(base)[i] = v;
  else if (dtype == kTypeF16)
    static_cast<__half*>(base)[i] = __float2half_rn(v);
  else
    static_cast<__nv_bfloat16*>(base)[i] = __float2bfloat16_rn(v);
}

// One CTA per (query head, query token): each of its warps takes every fourth position with its own
// running maximum and sum, E = D / 32 dimensions a lane, and the CTA joins the four.
constexpr int kWarps = 4;

template <int E>
__global__ void __launch_bounds__(kWarps * 32) kv4_attention_kernel(Kv4AttentionParams p, int dtype) {
  constexpr int D = 32 * E;
  __shared__ float s_m[kWarps], s_l[kWarps], s_acc[kWarps][D];
  const Kv4View& c = p.cache;
  const int head = blockIdx.y, token = blockIdx.x, kv_head = head / (p.q_heads / c.kv_heads);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int b = token, first = token, n = 1;
  if (p.query_start) {
    int lo = 0, hi = p.batch;  // the last sequence that starts at or before the token
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (p.query_start[mid] <= token) lo = mid;
      else hi = mid;
    }
    b = lo;
    first = max(p.query_start[b], 0);
    n = min(p.query_start[b + 1], p.tokens) - first;
    if (token < first || token >= first + n) return;  // of no sequence: left as it was
  }
  const int bs = 1 << c.shift;
  const long long reach = (long long)p.max_blocks << c.shift;
  const long long kv = min((long long)max(p.kv_lens[b], 0), reach);
  const long long sees = min(kv, (long long)p.kv_lens[b] - n + (token - first) + 1);
  float q[E], acc[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = load_any(p.q, token * p.q_stride + (long long)head * D + lane * E + e, dtype);
    acc[e] = 0.f;
  }
  const int g = lane * E / c.group, ng = D / c.group;
  for (long long t = warp; t < sees; t += kWarps) {
    const long long row = kv4_row(c, p.block_tables[(size_t)b * p.max_blocks + (t >> c.shift)], kv_head,
                                  (int)(t & (bs - 1)));
    if (row < 0) continue;
    float k[E], v[E];
    const uint32_t ks = c.k_scales[row * ng + g], vs = c.v_scales[row * ng + g];
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      const long long at = row * (D / 2) + (lane * E + e) / 2;
      const uint8_t kb = c.k_codes[at], vb = c.v_codes[at];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        k[e + i] = fmaf((float)(kb >> (4 * i) & 15), __half2float(__ushort_as_half((unsigned short)ks)),
                        __half2float(__ushort_as_half((unsigned short)(ks >> 16))));
        v[e + i] = fmaf((float)(vb >> (4 * i) & 15), __half2float(__ushort_as_half((unsigned short)vs)),
                        __half2float(__ushort_as_half((unsigned short)(vs >> 16))));
      }
    }
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s = fmaf(q[e], k[e], s);
    for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    s *= p.scale;
    const float nm = fmaxf(m, s), f = expf(m - nm), w = expf(s - nm);
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = acc[e] * f + w * v[e];
    l = l * f + w;
    m = nm;
  }
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) s_acc[warp][lane * E + e] = acc[e];
  __syncthreads();
  for (int d = threadIdx.x; d < D; d += kWarps * 32) {
    float top = -INFINITY, sum = 0.f, o = 0.f;
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w]);
    for (int w = 0; w < kWarps; ++w) {
      if (s_l[w] == 0.f) continue;
      const float f = expf(s_m[w] - top);
      sum += s_l[w] * f;
      o += s_acc[w][d] * f;
    }
    store_any(p.o, token * p.o_stride + (long long)head * D + d, dtype, sum == 0.f ? 0.f : o / sum);
  }
}

}  // namespace

size_t kv4_attention_workspace(int, int) { return 256; }

cudaError_t launch_kv4_attention(const Kv4AttentionParams& p, int dtype, int, cudaStream_t st) {
  const dim3 grid((unsigned)p.tokens, (unsigned)p.q_heads);
  switch (p.cache.head_dim) {
    case 64: kv4_attention_kernel<2><<<grid, kWarps * 32, 0, st>>>(p, dtype); break;
    case 128: kv4_attention_kernel<4><<<grid, kWarps * 32, 0, st>>>(p, dtype); break;
    default: kv4_attention_kernel<8><<<grid, kWarps * 32, 0, st>>>(p, dtype); break;
  }
  return cudaGetLastError();
}

}  // namespace tk
