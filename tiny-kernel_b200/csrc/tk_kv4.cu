// tk_kv4.cu -- the operators that feed the 4-bit key/value cache: block tables and slots of a step,
// per-head norms with the position rotation, quantised writes and reads.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cstdint>

#include "tk_kv4.h"

namespace tk {
namespace {

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
// 32 bytes).
template <class T, int E>
__device__ __forceinline__ void load_f32(const T* src, bool vec, float (&v)[E]) {
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
__device__ __forceinline__ void store_f32(T* dst, bool vec, const float (&v)[E]) {
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

// ---- block tables and slots ----------------------------------------------------------------------
//
// Two exclusive prefix sums over the requests (tokens, pages to take) give every token its request
// and every page its place in the free list.  Every CTA computes the sums itself: 8 bytes a request
// from L2, against a second launch or a wait between CTAs.  A thread owns a run of consecutive
// requests and only the sums at the runs' starts are kept, so the batch has no limit; a token finds
// its run by binary search and walks it.  No atomics: the last CTA writes what is per request and
// counts the tokens without a slot on its own.
constexpr int kSlotsThreads = 256;
constexpr int kSlotsTokens = 4;  // consecutive tokens of a thread: one search, 16-byte stores

__device__ __forceinline__ long long block_exclusive_scan(long long v, long long* warp_sums,
                                                          long long* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long inc = v;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const long long o = __shfl_up_sync(0xffffffffu, inc, off);
    if (lane >= off) inc += o;
  }
  __syncthreads();  // the sums of an earlier scan have been read
  if (lane == 31) warp_sums[warp] = inc;
  __syncthreads();
  long long before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kSlotsThreads / 32; ++w) {
    const long long s = warp_sums[w];
    if (w < warp) before += s;
    all += s;
  }
  *total = all;
  return before + inc - v;
}

// The last run whose sum is at most `at`.
__device__ __forceinline__ int find_run(const long long* sums, long long at) {
  int lo = 0;
#pragma unroll
  for (int step = kSlotsThreads / 2; step > 0; step >>= 1)
    if (lo + step < kSlotsThreads && sums[lo + step] <= at) lo += step;
  return lo;
}

// A request with the sums at its start.
struct SlotsCursor {
  int r;
  long long start, first;  // tokens and pages of the requests before it
  SlotsRequest req;
  __device__ void at(const SlotsParams& p) {
    req = slots_request(p.context_lens[r], p.query_lens[r], start, p.shift, p.max_blocks, p.max_tokens);
  }
  __device__ void next(const SlotsParams& p) {
    start += slots_wanted(p.context_lens[r], p.query_lens[r]);
    first += req.need - req.have;
    ++r;
  }
};

__global__ void __launch_bounds__(kSlotsThreads) paged_slots_kernel(SlotsParams p) {
  __shared__ long long s_start[kSlotsThreads], s_first[kSlotsThreads], s_warp[kSlotsThreads / 32];
  const int tid = threadIdx.x;
  const int per = (p.batch + kSlotsThreads - 1) / kSlotsThreads;
  const int r0 = min((long long)p.batch, (long long)tid * per), r1 = min(p.batch, r0 + per);
  const int begin = p.free_range[0], end = p.free_range[1];

  long long sum = 0, asked, taken;
  for (int r = r0; r < r1; ++r) sum += slots_wanted(p.context_lens[r], p.query_lens[r]);
  const long long start0 = block_exclusive_scan(sum, s_warp, &asked);
  SlotsCursor c{r0, start0, 0, {}};
  while (c.r < r1) {
    c.at(p);
    c.next(p);
  }
  const long long first0 = block_exclusive_scan(c.first, s_warp, &taken);
  s_start[tid] = start0;
  s_first[tid] = first0;
  __syncthreads();
  const int tokens = (int)min(asked, (long long)p.max_tokens);
  const int bs1 = (1 << p.shift) - 1;

  const bool wide = ((reinterpret_cast<uintptr_t>(p.positions) | reinterpret_cast<uintptr_t>(p.slots)) & 15) == 0;
  for (long long t0 = ((long long)blockIdx.x * kSlotsThreads + tid) * kSlotsTokens; t0 < p.max_tokens;
       t0 += (long long)gridDim.x * kSlotsThreads * kSlotsTokens) {
    int pos[kSlotsTokens], slot[kSlotsTokens];
    if (t0 < tokens) {
      const int run = find_run(s_start, t0);
      c = {run * per, s_start[run], s_first[run], {}};
      c.at(p);
    }
#pragma unroll
    for (int i = 0; i < kSlotsTokens; ++i) {
      const long long t = t0 + i;
      pos[i] = slot[i] = -1;
      if (t >= tokens) continue;
      while (t >= c.start + c.req.q) {  // t < tokens: a later request holds it
        c.next(p);
        c.at(p);
      }
      pos[i] = c.req.ctx + (int)(t - c.start);
      const int page = pos[i] >> p.shift;
      if (page >= p.max_blocks) continue;
      int* entry = p.block_tables + (size_t)c.r * p.max_blocks + page;
      int id;
      if (page < c.req.have) {
        id = *entry;
        if (id >= p.num_blocks) id = -1;
      } else {
        id = slots_new_block(p.free_blocks, begin, end, c.first + page - c.req.have, p.num_blocks);
        if ((pos[i] & bs1) == 0) *entry = id;  // a new page's first token is of this step
      }
      if (id >= 0) slot[i] = (id << p.shift) + (pos[i] & bs1);
    }
    if (wide && t0 + kSlotsTokens <= p.max_tokens) {
      *reinterpret_cast<int4*>(p.positions + t0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
      *reinterpret_cast<int4*>(p.slots + t0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
    } else {
#pragma unroll
      for (int i = 0; i < kSlotsTokens; ++i)
        if (t0 + i < p.max_tokens) {
          p.positions[t0 + i] = pos[i];
          p.slots[t0 + i] = slot[i];
        }
    }
  }

  if (blockIdx.x != gridDim.x - 1) return;
  long long without = 0;
  c = {r0, start0, first0, {}};
  while (c.r < r1) {
    c.at(p);
    const SlotsRequest& q = c.req;
    p.kv_lens[c.r] = q.ctx + q.q;
    p.query_start[c.r] = (int)min(c.start, (long long)p.max_tokens);
    if (q.q > 0 && (q.ctx & bs1) && (q.ctx >> p.shift) < p.max_blocks) {  // the page it has begun
      const int id = p.block_tables[(size_t)c.r * p.max_blocks + (q.ctx >> p.shift)];
      if (id < 0 || id >= p.num_blocks) without += slots_tokens_in(q, q.ctx >> p.shift, p.shift);
    }
    const long long reach = max((long long)p.max_blocks << p.shift, (long long)q.ctx);
    without += max(0ll, (long long)q.ctx + q.q - reach);
    c.next(p);
  }
  for (long long a = tid; a < taken; a += kSlotsThreads) {  // pages that the pool did not have
    if (slots_new_block(p.free_blocks, begin, end, a, p.num_blocks) >= 0) continue;
    const int run = find_run(s_first, a);
    c = {run * per, s_start[run], s_first[run], {}};
    c.at(p);
    while (a >= c.first + c.req.need - c.req.have) {
      c.next(p);
      c.at(p);
    }
    without += slots_tokens_in(c.req, c.req.have + (int)(a - c.first), p.shift);
  }
  long long all;
  block_exclusive_scan(without, s_warp, &all);
  if (tid == 0) {
    p.query_start[p.batch] = tokens;
    p.counts[0] = tokens;
    p.counts[1] = (int)taken;
    p.counts[2] = (int)all;
    const long long first = begin > 0 ? begin : 0;
    p.counts[3] = (int)max(first, min(first + taken, (long long)end));
  }
}

// ---- norms of queries and keys, and the rotation -------------------------------------------------
//
// y = x * rsqrt(mean(x^2) + eps) * w over a head, then for each pair (a, b) of the rotated part
// (a cos - b sin, b cos + a sin).  Everything in f32, one rounding at the store.

struct QkRow {
  int which, head;  // 0: queries, 1: keys
};
__device__ __forceinline__ QkRow qk_row(const QkNormRopeParams& p, int head) {
  return head < p.heads[0] ? QkRow{0, head} : QkRow{1, head - p.heads[0]};
}

// LPH lanes hold a head, E consecutive values each (16 or 32 bytes); the pair of a value lies
// rot_dim / 2 values on, a multiple of E: the same place in another lane.
template <class T, int E, int LPH>
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(QkNormRopeParams p, int vec_in, int vec_out,
                                                           int heads_per_group) {
  const int lane = threadIdx.x & 31, l = lane % LPH;
  const int heads = p.heads[0] + p.heads[1];
  const int parts = (heads + heads_per_group - 1) / heads_per_group;
  const long long group = ((long long)blockIdx.x * blockDim.x + threadIdx.x) / LPH;
  const long long token = group / parts;
  const int h0 = (int)(group % parts) * heads_per_group, h1 = min(heads, h0 + heads_per_group);
  const int half = p.rot_dim / 2;
  const int pos = token < p.tokens ? p.positions[token] : -1;
  const bool on = pos >= 0 && pos < p.max_pos;
  if (!__any_sync(0xffffffffu, on)) return;

  // what the lane's values are turned by (1, 0 past rot_dim), and the lane of their pairs
  float c[E], s[E];
  int src = lane;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int i = l * E + e;
    const int j = p.interleaved ? i / 2 : (i < half ? i : i - half);
    const bool turned = on && i < p.rot_dim;
    c[e] = turned ? p.cos_cache[(size_t)pos * half + j] : 1.f;
    s[e] = turned ? p.sin_cache[(size_t)pos * half + j] : 0.f;
    if (p.interleaved ? (i & 1) == 0 : i < half) s[e] = -s[e];
  }
  if (!p.interleaved && l * E < p.rot_dim) src = l * E < half ? lane + half / E : lane - half / E;

  for (int h = h0; h < h0 + heads_per_group; ++h) {  // the same count in every lane of the warp
    const bool mine = on && h < h1;
    const QkRow r = qk_row(p, min(h, heads - 1));
    float y[E];
#pragma unroll
    for (int e = 0; e < E; ++e) y[e] = 0.f;
    if (mine)
      load_f32<T, E>(static_cast<const T*>(p.x[r.which]) + token * p.in_stride[r.which] +
                         (long long)r.head * p.head_dim + l * E,
                     vec_in, y);
    const float* w = p.weight[r.which];
    if (w) {
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) ss = fmaf(y[e], y[e], ss);
#pragma unroll
      for (int off = LPH / 2; off > 0; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
      const float inv = rsqrtf(ss / (float)p.head_dim + p.eps);
#pragma unroll
      for (int e = 0; e < E; ++e) y[e] = y[e] * inv * __ldg(w + l * E + e);
    }
    // a value past rot_dim is its own pair, with sine 0: it must not meet an infinity times 0
    float z[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float other = p.interleaved ? y[e ^ 1] : __shfl_sync(0xffffffffu, y[e], src);
      z[e] = l * E + e < p.rot_dim ? y[e] * c[e] + other * s[e] : y[e];
    }
    if (mine)
      store_f32<T, E>(static_cast<T*>(p.out[r.which]) + token * p.out_stride[r.which] +
                          (long long)r.head * p.head_dim + l * E,
                      vec_out, z);
  }
}

// Any even head_dim up to kQkMaxDim: a warp per head, the normalised row in shared memory.
constexpr int kQkMaxDim = 1024;
constexpr int kQkWarps = 4;

template <class T>
__global__ void __launch_bounds__(kQkWarps * 32) qk_norm_rope_any_kernel(QkNormRopeParams p) {
  extern __shared__ float s_rows[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, d = p.head_dim, half = p.rot_dim / 2;
  float* row = s_rows + warp * d;
  const int heads = p.heads[0] + p.heads[1];
  const long long unit = (long long)blockIdx.x * kQkWarps + warp;
  if (unit >= (long long)p.tokens * heads) return;
  const long long token = unit / heads;
  const int pos = p.positions[token];
  if (pos < 0 || pos >= p.max_pos) return;
  const QkRow r = qk_row(p, (int)(unit % heads));
  const T* x = static_cast<const T*>(p.x[r.which]) + token * p.in_stride[r.which] + (long long)r.head * d;
  T* out = static_cast<T*>(p.out[r.which]) + token * p.out_stride[r.which] + (long long)r.head * d;
  const float* w = p.weight[r.which];
  float ss = 0.f;
  for (int i = lane; i < d; i += 32) {
    const float v = to_f32(x[i]);
    row[i] = v;
    ss = fmaf(v, v, ss);
  }
  if (w) {
    for (int off = 16; off > 0; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
    const float inv = rsqrtf(ss / (float)d + p.eps);
    for (int i = lane; i < d; i += 32) row[i] = row[i] * inv * w[i];
  }
  __syncwarp();
  for (int i = lane; i < d; i += 32) {
    float z = row[i];
    if (i < p.rot_dim) {
      const int j = p.interleaved ? i / 2 : (i < half ? i : i - half);
      const bool first = p.interleaved ? (i & 1) == 0 : i < half;
      const float other = row[p.interleaved ? i ^ 1 : (first ? i + half : i - half)];
      const float c = p.cos_cache[(size_t)pos * half + j], s = p.sin_cache[(size_t)pos * half + j];
      z = first ? z * c - other * s : z * c + other * s;
    }
    out[i] = from_f32<T>(z);
  }
}

template <class T, int E, int LPH>
cudaError_t qk_launch_vec(const QkNormRopeParams& p, bool vec_in, bool vec_out, int sm_count, cudaStream_t st) {
  const int heads = p.heads[0] + p.heads[1];
  const int hpg = 1;
  (void)sm_count;
  const long long groups = (long long)p.tokens * ((heads + hpg - 1) / hpg);
  const long long blocks = (groups * LPH + 255) / 256;
  qk_norm_rope_kernel<T, E, LPH><<<(unsigned)blocks, 256, 0, st>>>(p, vec_in, vec_out, hpg);
  return cudaGetLastError();
}

template <class T>
cudaError_t qk_launch(const QkNormRopeParams& p, int sm_count, cudaStream_t st) {
  const int size = (int)sizeof(T);
  bool vec_in = true, vec_out = true;
  for (int i = 0; i < 2; ++i) {
    if (p.heads[i] == 0) continue;
    vec_in = vec_in && reinterpret_cast<uintptr_t>(p.x[i]) % 16 == 0 && p.in_stride[i] * size % 16 == 0;
    vec_out = vec_out && reinterpret_cast<uintptr_t>(p.out[i]) % 16 == 0 && p.out_stride[i] * size % 16 == 0;
  }
  constexpr int E = 16 / (int)sizeof(T);  // 16 bytes a lane
  const int half = p.rot_dim / 2;
  const int e = p.head_dim == 256 ? 8 : E;
  if (p.interleaved || half % e == 0) {
    if (p.head_dim == 64) return qk_launch_vec<T, E, 64 / E>(p, vec_in, vec_out, sm_count, st);
    if (p.head_dim == 128) return qk_launch_vec<T, E, 128 / E>(p, vec_in, vec_out, sm_count, st);
    if (p.head_dim == 256) return qk_launch_vec<T, 8, 32>(p, vec_in, vec_out, sm_count, st);
  }
  const long long units = (long long)p.tokens * (p.heads[0] + p.heads[1]);
  qk_norm_rope_any_kernel<T><<<(unsigned)((units + kQkWarps - 1) / kQkWarps), kQkWarps * 32,
                               kQkWarps * p.head_dim * sizeof(float), st>>>(p);
  return cudaGetLastError();
}

// ---- quantised writes and reads ------------------------------------------------------------------
//
// A group of G values: offset m = f16(min), scale s = f16((max - min) / 15), codes
// clamp(rint((x - m) / s), 0, 15) with the true quotient rounded to the nearest, ties to even.  The
// quotient in f32 is off by under 2e-6 (two roundings of 2^-24 of at most 15.01), so only one that
// close to a tie is settled in 64 bits; the two 64-bit operations a group that make s round right
// are 1/64 of the work.  8 values a lane: one 16-byte load (f16, bf16) or two (f32), one 32-bit
// store of codes; a group is 8 or 16 lanes.
constexpr int kKv4Lane = 8;

__device__ __forceinline__ int kv4_code(float x, float m, float s) {
  const float q = __fdiv_rn(x - m, s);
  float c = rintf(q);
  if (fabsf(fabsf(q - c) - 0.5f) < 4e-6f) c = (float)rint(((double)x - (double)m) / (double)s);
  return (int)fminf(fmaxf(c, 0.f), 15.f);
}

template <class T>
__global__ void __launch_bounds__(256) kv4_append_kernel(Kv4View c, const T* __restrict__ k,
                                                         const T* __restrict__ v,
                                                         const int* __restrict__ slots, int tokens,
                                                         long long k_stride, long long v_stride, int vec) {
  const int lanes = c.head_dim / kKv4Lane;  // 8, 16 or 32 lanes a row
  const long long thread = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  const int l = (int)(thread % lanes);
  long long unit = thread / lanes;  // (token, keys or values, head)
  const int head = (int)(unit % c.kv_heads);
  unit /= c.kv_heads;
  const bool values = unit & 1;
  const long long token = unit >> 1;
  const int slot = token < tokens ? slots[token] : -1;
  const long long row = kv4_slot_row(c, slot, head);
  float x[kKv4Lane];
#pragma unroll
  for (int e = 0; e < kKv4Lane; ++e) x[e] = 0.f;
  if (row >= 0)
    load_f32<T, kKv4Lane>((values ? v + token * v_stride : k + token * k_stride) + head * c.head_dim +
                              l * kKv4Lane,
                          vec, x);
  // min and max pass over a NaN, and an infinity has none of the two: 0 * x is 0 or NaN, and its
  // sum makes the group's offset and scale NaN wherever a value is not finite
  float lo = x[0], hi = x[0], odd = 0.f;
#pragma unroll
  for (int e = 0; e < kKv4Lane; ++e) {
    lo = fminf(lo, x[e]);
    hi = fmaxf(hi, x[e]);
    odd = fmaf(x[e], 0.f, odd);
  }
  for (int off = c.group / kKv4Lane / 2; off > 0; off >>= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, off));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, off));
    odd += __shfl_xor_sync(0xffffffffu, odd, off);
  }
  if (row < 0) return;
  // finite values past f16 saturate
  const float range = (float)(((double)hi - (double)lo) / 15.0);
  const __half hs = __float2half_rn(fminf(range, 65504.f) + odd);
  const __half hm = __float2half_rn(fminf(fmaxf(lo, -65504.f), 65504.f) + odd);
  const float s = __half2float(hs), m = __half2float(hm);
  uint32_t word = 0;
  if (s > 0.f) {
#pragma unroll
    for (int e = 0; e < kKv4Lane; ++e) word |= (uint32_t)kv4_code(x[e], m, s) << (4 * e);
  }
  uint8_t* codes = values ? c.v_codes : c.k_codes;
  uint32_t* scales = values ? c.v_scales : c.k_scales;
  *reinterpret_cast<uint32_t*>(codes + row * (c.head_dim / 2) + l * (kKv4Lane / 2)) = word;
  const int lane_of_group = c.group / kKv4Lane;
  if (l % lane_of_group == 0)
    scales[row * (c.head_dim / c.group) + l / lane_of_group] =
        (uint32_t)__half_as_ushort(hs) | (uint32_t)__half_as_ushort(hm) << 16;
}

template <class T>
__global__ void __launch_bounds__(256) kv4_gather_kernel(Kv4View c, T* __restrict__ k, T* __restrict__ v,
                                                         const int* __restrict__ slots, int tokens,
                                                         long long k_stride, long long v_stride, int vec) {
  const int lanes = c.head_dim / kKv4Lane;
  const long long thread = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  const int l = (int)(thread % lanes);
  long long unit = thread / lanes;
  const int head = (int)(unit % c.kv_heads);
  unit /= c.kv_heads;
  const bool values = unit & 1;
  const long long token = unit >> 1;
  if (token >= tokens) return;
  const long long row = kv4_slot_row(c, slots[token], head);
  if (row < 0) return;
  const uint8_t* codes = values ? c.v_codes : c.k_codes;
  const uint32_t* scales = values ? c.v_scales : c.k_scales;
  const uint32_t word = *reinterpret_cast<const uint32_t*>(codes + row * (c.head_dim / 2) + l * (kKv4Lane / 2));
  const uint32_t pair = scales[row * (c.head_dim / c.group) + l * kKv4Lane / c.group];
  const float s = __half2float(__ushort_as_half((unsigned short)pair));
  const float m = __half2float(__ushort_as_half((unsigned short)(pair >> 16)));
  float x[kKv4Lane];
#pragma unroll
  for (int e = 0; e < kKv4Lane; ++e) x[e] = fmaf((float)(word >> (4 * e) & 15u), s, m);
  store_f32<T, kKv4Lane>((values ? v + token * v_stride : k + token * k_stride) + head * c.head_dim +
                             l * kKv4Lane,
                         vec, x);
}

template <class T>
bool rows_vec(const void* k, const void* v, long long k_stride, long long v_stride) {
  return (reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % 16 == 0 &&
         k_stride * (long long)sizeof(T) % 16 == 0 && v_stride * (long long)sizeof(T) % 16 == 0;
}

unsigned kv4_blocks(const Kv4View& c, int tokens) {
  return (unsigned)(((long long)tokens * 2 * c.kv_heads * (c.head_dim / kKv4Lane) + 255) / 256);
}

template <class T>
cudaError_t append(const Kv4View& c, const void* k, const void* v, const int* slots, int tokens,
                   long long k_stride, long long v_stride, cudaStream_t st) {
  kv4_append_kernel<T><<<kv4_blocks(c, tokens), 256, 0, st>>>(
      c, static_cast<const T*>(k), static_cast<const T*>(v), slots, tokens, k_stride, v_stride,
      rows_vec<T>(k, v, k_stride, v_stride));
  return cudaGetLastError();
}

template <class T>
cudaError_t gather(const Kv4View& c, void* k, void* v, const int* slots, int tokens, long long k_stride,
                   long long v_stride, cudaStream_t st) {
  kv4_gather_kernel<T><<<kv4_blocks(c, tokens), 256, 0, st>>>(
      c, static_cast<T*>(k), static_cast<T*>(v), slots, tokens, k_stride, v_stride,
      rows_vec<T>(k, v, k_stride, v_stride));
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_paged_slots(const SlotsParams& p, int sm_count, cudaStream_t st) {
  const long long per = kSlotsThreads * kSlotsTokens;
  const long long blocks = std::max(1ll, std::min((p.max_tokens + per - 1) / per, (long long)sm_count * 2));
  paged_slots_kernel<<<(unsigned)blocks, kSlotsThreads, 0, st>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_qk_norm_rope(const QkNormRopeParams& p, int dtype, int sm_count, cudaStream_t st) {
  switch (dtype) {
    case kTypeF32: return qk_launch<float>(p, sm_count, st);
    case kTypeF16: return qk_launch<__half>(p, sm_count, st);
    default: return qk_launch<__nv_bfloat16>(p, sm_count, st);
  }
}

cudaError_t launch_kv4_append(const Kv4View& c, const void* k, const void* v, const int* slots, int tokens,
                              long long k_stride, long long v_stride, int dtype, cudaStream_t st) {
  switch (dtype) {
    case kTypeF32: return append<float>(c, k, v, slots, tokens, k_stride, v_stride, st);
    case kTypeF16: return append<__half>(c, k, v, slots, tokens, k_stride, v_stride, st);
    default: return append<__nv_bfloat16>(c, k, v, slots, tokens, k_stride, v_stride, st);
  }
}

cudaError_t launch_kv4_gather(const Kv4View& c, void* k, void* v, const int* slots, int tokens,
                              long long k_stride, long long v_stride, int dtype, cudaStream_t st) {
  switch (dtype) {
    case kTypeF32: return gather<float>(c, k, v, slots, tokens, k_stride, v_stride, st);
    case kTypeF16: return gather<__half>(c, k, v, slots, tokens, k_stride, v_stride, st);
    default: return gather<__nv_bfloat16>(c, k, v, slots, tokens, k_stride, v_stride, st);
  }
}

}  // namespace tk
