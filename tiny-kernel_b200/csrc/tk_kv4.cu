// tk_kv4.cu -- the operators that feed the 4-bit key/value cache: block tables and slots of a step,
// per-head norms with the position rotation, quantised writes and reads.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "tk_kv4.h"

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

// E/2 elements at src and E/2 at src + next.  vec: both on the boundary of their 8 or 16 bytes.
template <class T, int E>
__device__ __forceinline__ void load_halves(const T* src, int next, bool vec, float (&v)[E]) {
  constexpr int H = E / 2;
  using V = typename std::conditional<H * sizeof(T) == 16, uint4, uint2>::type;
  if (vec) {
    V raw[2] = {*reinterpret_cast<const V*>(src), *reinterpret_cast<const V*>(src + next)};
    const T* e = reinterpret_cast<const T*>(raw);
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = to_f32(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = to_f32(src[(i / H) * next + i % H]);
  }
}
template <class T, int E>
__device__ __forceinline__ void store_halves(T* dst, int next, bool vec, const float (&v)[E]) {
  constexpr int H = E / 2;
  using V = typename std::conditional<H * sizeof(T) == 16, uint4, uint2>::type;
  if (vec) {
    V raw[2];
    T* e = reinterpret_cast<T*>(raw);
#pragma unroll
    for (int i = 0; i < E; ++i) e[i] = from_f32<T>(v[i]);
    *reinterpret_cast<V*>(dst) = raw[0];
    *reinterpret_cast<V*>(dst + next) = raw[1];
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) dst[(i / H) * next + i % H] = from_f32<T>(v[i]);
  }
}

// ---- block tables and slots ----------------------------------------------------------------------
//
// Two exclusive prefix sums over the requests (tokens, pages to take) give every token its request
// and every page its place in the free list.  Every CTA computes the sums itself: 8 bytes a request
// from L2, against a second launch or a wait between CTAs.  A thread owns a run of consecutive
// requests and only the sums at the runs' starts are kept, so the batch has no limit; a token finds
// its run by binary search and walks it.  No atomics: one CTA (the only
// one of a small step) writes what is per request and counts the tokens without a slot.
constexpr int kSlotsThreads = 256;

// Exclusive sums of two values a thread; totals in all[2].
struct SlotsSums {
  long long tokens, pages;
};
__device__ __forceinline__ SlotsSums block_exclusive_scan(SlotsSums v, SlotsSums* warp_sums, SlotsSums* all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  SlotsSums inc = v;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const long long t = __shfl_up_sync(0xffffffffu, inc.tokens, off), g = __shfl_up_sync(0xffffffffu, inc.pages, off);
    if (lane >= off) {
      inc.tokens += t;
      inc.pages += g;
    }
  }
  __syncthreads();  // the sums of an earlier scan have been read
  if (lane == 31) warp_sums[warp] = inc;
  __syncthreads();
  SlotsSums before{0, 0}, total{0, 0};
#pragma unroll
  for (int w = 0; w < kSlotsThreads / 32; ++w) {
    const SlotsSums s = warp_sums[w];
    if (w < warp) before = {before.tokens + s.tokens, before.pages + s.pages};
    total = {total.tokens + s.tokens, total.pages + s.pages};
  }
  *all = total;
  return {before.tokens + inc.tokens - v.tokens, before.pages + inc.pages - v.pages};
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

// TOK: consecutive tokens of a thread (4: one search and 16-byte stores for four).
template <int TOK>
__global__ void __launch_bounds__(kSlotsThreads) paged_slots_kernel(SlotsParams p) {
  __shared__ long long s_start[kSlotsThreads], s_first[kSlotsThreads];
  __shared__ SlotsSums s_warp[kSlotsThreads / 32];
  after_previous();
  const int tid = threadIdx.x;
  const bool alone = gridDim.x == 1, requests = blockIdx.x == gridDim.x - 1;
  const int per = (p.batch + kSlotsThreads - 1) / kSlotsThreads;
  const int r0 = (int)min((long long)p.batch, (long long)tid * per), r1 = min(p.batch, r0 + per);
  const int begin = p.free_range[0], end = p.free_range[1];
  const int bs1 = (1 << p.shift) - 1;

  // Both sums at once, as if all tokens had room; if they have not, the pages are summed again.
  SlotsSums sum{0, 0}, all;
  for (int r = r0; r < r1; ++r) {
    const int ctx = p.context_lens[r], q = p.query_lens[r];
    const SlotsRequest x = slots_request(ctx, q, -0x7fffffffffffll, p.shift, p.max_blocks, p.max_tokens);
    sum.tokens += slots_wanted(ctx, q);
    sum.pages += x.need - x.have;
  }
  SlotsSums at0 = block_exclusive_scan(sum, s_warp, &all);
  const long long asked = all.tokens, start0 = at0.tokens;
  SlotsCursor c;
  if (asked > p.max_tokens) {
    c = {r0, start0, 0, {}};
    while (c.r < r1) {
      c.at(p);
      c.next(p);
    }
    at0 = block_exclusive_scan({0, c.first}, s_warp, &all);
  }
  const long long first0 = at0.pages, taken = all.pages;
  s_start[tid] = start0;
  s_first[tid] = first0;
  __syncthreads();
  const int tokens = (int)min(asked, (long long)p.max_tokens);

  const bool wide = ((reinterpret_cast<uintptr_t>(p.positions) | reinterpret_cast<uintptr_t>(p.slots)) & 15) == 0;
  const int token_ctas = alone ? 1 : gridDim.x - 1;
  for (long long t0 = ((long long)blockIdx.x * kSlotsThreads + tid) * TOK;
       t0 < p.max_tokens && (alone || !requests); t0 += (long long)token_ctas * kSlotsThreads * TOK) {
    int pos[TOK], slot[TOK];
    if (t0 < tokens) {
      const int run = find_run(s_start, t0);
      c = {run * per, s_start[run], s_first[run], {}};
      c.at(p);
    }
#pragma unroll
    for (int i = 0; i < TOK; ++i) {
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
    bool stored = false;
    if constexpr (TOK == 4) {
      if (wide && t0 + TOK <= p.max_tokens) {
        *reinterpret_cast<int4*>(p.positions + t0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
        *reinterpret_cast<int4*>(p.slots + t0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
        stored = true;
      }
    }
    if (!stored) {
#pragma unroll
      for (int i = 0; i < TOK; ++i)
        if (t0 + i < p.max_tokens) {
          p.positions[t0 + i] = pos[i];
          p.slots[t0 + i] = slot[i];
        }
    }
  }

  if (!requests) return;
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
  constexpr int kIds = 16;  // reads in flight of a thread
  const long long free0 = begin > 0 ? begin : 0;
  for (long long a0 = tid; a0 < taken; a0 += kSlotsThreads * kIds) {  // pages that the pool did not have
    int id[kIds];
#pragma unroll
    for (int i = 0; i < kIds; ++i) {  // read without a branch, some valid place at least
      const long long x = free0 + a0 + i * kSlotsThreads;
      id[i] = free0 < end ? p.free_blocks[x < end ? x : free0] : -1;
    }
    const long long left = end - free0 - a0;  // of the list from this place
    bool bad = false;
#pragma unroll
    for (int i = 0; i < kIds; ++i)
      bad = bad || (unsigned)id[i] >= (unsigned)p.num_blocks || i * kSlotsThreads >= left;
    if (!bad) continue;
#pragma unroll 1
    for (int i = 0; i < kIds; ++i) {
      const long long a = a0 + (long long)i * kSlotsThreads;
      if (a >= taken || slots_new_block(p.free_blocks, begin, end, a, p.num_blocks) >= 0) continue;
      const int run = find_run(s_first, a);
      c = {run * per, s_start[run], s_first[run], {}};
      c.at(p);
      while (a >= c.first + c.req.need - c.req.have) {
        c.next(p);
        c.at(p);
      }
      without += slots_tokens_in(c.req, c.req.have + (int)(a - c.first), p.shift);
    }
  }
  block_exclusive_scan({without, 0}, s_warp, &all);
  if (tid == 0) {
    p.query_start[p.batch] = tokens;
    p.counts[0] = tokens;
    p.counts[1] = (int)taken;
    p.counts[2] = (int)all.tokens;
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

// Up to LPH lanes hold a head, E values each (16 or 32 bytes); a group of LPH lanes takes HB queries or
// keys of a token, so that weights and angles are read once and HB loads are in flight: bound by HBM.
//   kHalves (the whole head turns, by halves): a lane holds E/2 consecutive values of each half, and so
//     both values of a pair;
//   kPairs (interleaved): E consecutive values;
//   kPart (a part of the head turns, by halves): E consecutive values; the pair of one lies rot_dim / 2
//     values on, a multiple of E: the same place in another lane.
// EXACT: head_dim is E * LPH, and else less.
enum QkMode { kHalves, kPairs, kPart };

template <class T, int E, int LPH, int HB, int MODE, bool EXACT>
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(QkNormRopeParams p, int vec_in, int vec_out, int vec_turn) {
  constexpr int H = E / 2;
  after_previous();
  const int D = EXACT ? E * LPH : p.head_dim;
  const int lane = threadIdx.x & 31, l = lane % LPH;
  const bool holds = EXACT || l * E < D;
  const int q_parts = (p.heads[0] + HB - 1) / HB, parts = q_parts + (p.heads[1] + HB - 1) / HB;
  const unsigned group = (unsigned)(((long long)blockIdx.x * blockDim.x + threadIdx.x) / LPH);  // below 2^31
  const int token = (int)(group / (unsigned)parts), part = (int)(group - (unsigned)token * parts);
  const int which = part >= q_parts, h0 = (which ? part - q_parts : part) * HB, heads = p.heads[which];
  const int half = p.rot_dim / 2;
  const int pos = token < p.tokens ? p.positions[token] : -1;
  const bool on = pos >= 0 && pos < p.max_pos;
  if (!__any_sync(0xffffffffu, on)) return;

  float y[HB][E];
  const T* x = static_cast<const T*>(p.x[which]) + token * p.in_stride[which] + (long long)h0 * D;
#pragma unroll
  for (int i = 0; i < HB; ++i) {
#pragma unroll
    for (int e = 0; e < E; ++e) y[i][e] = 0.f;
    if (on && holds && h0 + i < heads) {
      if constexpr (MODE == kHalves)
        load_halves<T, E>(x + i * D + l * H, D / 2, vec_in, y[i]);
      else
        load_f32<T, E>(x + i * D + l * E, vec_in, y[i]);
    }
  }

  // what the lane's values are turned by (1, 0 past rot_dim), and the lane of their pairs
  constexpr int A = MODE == kPart ? E : H;
  float c[A], s[A];
  int src = lane;
#pragma unroll
  for (int e = 0; e < A; ++e) c[e] = 1.f, s[e] = 0.f;
  if (on && holds && (MODE == kHalves || l * E < p.rot_dim)) {
    const int j0 = MODE != kPart ? l * H : l * E < half ? l * E : l * E - half;
    const float* cp = p.cos_cache + (size_t)pos * half + j0;
    const float* sp = p.sin_cache + (size_t)pos * half + j0;
    if (vec_turn && (MODE != kPairs || l * E + E <= p.rot_dim)) {  // by pairs on 8-byte boundaries
#pragma unroll
      for (int e = 0; e < A; e += 2) {
        const float2 cv = *reinterpret_cast<const float2*>(cp + e), sv = *reinterpret_cast<const float2*>(sp + e);
        c[e] = cv.x, c[e + 1] = cv.y;
        s[e] = sv.x, s[e + 1] = sv.y;
      }
    } else {
#pragma unroll
      for (int e = 0; e < A; ++e)
        if (j0 + e < half) {
          c[e] = cp[e];
          s[e] = sp[e];
        }
    }
    if constexpr (MODE == kPart) {
#pragma unroll
      for (int e = 0; e < A; ++e)
        if (l * E < half) s[e] = -s[e];
      src = l * E < half ? lane + half / E : lane - half / E;
    }
  }
  const float* wp = p.weight[which];
  float w[E];
#pragma unroll
  for (int e = 0; e < E; ++e)
    w[e] = wp && holds ? wp[MODE == kHalves ? (e / H) * (D / 2) + l * H + e % H : l * E + e] : 1.f;

  T* out = static_cast<T*>(p.out[which]) + token * p.out_stride[which] + (long long)h0 * D;
#pragma unroll
  for (int i = 0; i < HB; ++i) {
    if (p.weight[0] || p.weight[1]) {  // the same for all lanes: queries and keys may share a warp
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) ss = fmaf(y[i][e], y[i][e], ss);
#pragma unroll
      for (int off = LPH / 2; off > 0; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
      if (wp) {
        const float inv = rsqrtf(ss / (float)D + p.eps);
#pragma unroll
        for (int e = 0; e < E; ++e) y[i][e] = y[i][e] * inv * w[e];
      }
    }
    float z[E];
    if constexpr (MODE == kPart) {
      // a value past rot_dim stays: it must not meet an infinity times 0
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float other = __shfl_sync(0xffffffffu, y[i][e], src);
        z[e] = l * E < p.rot_dim ? y[i][e] * c[e] + other * s[e] : y[i][e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < H; ++e) {
        const int a = MODE == kHalves ? e : 2 * e, b = MODE == kHalves ? H + e : 2 * e + 1;
        const bool stays = MODE == kPairs && l * E + a >= p.rot_dim;
        z[a] = stays ? y[i][a] : y[i][a] * c[e] - y[i][b] * s[e];
        z[b] = stays ? y[i][b] : y[i][b] * c[e] + y[i][a] * s[e];
      }
    }
    if (on && holds && h0 + i < heads) {
      if constexpr (MODE == kHalves)
        store_halves<T, E>(out + i * D + l * H, D / 2, vec_out, z);
      else
        store_f32<T, E>(out + i * D + l * E, vec_out, z);
    }
  }
}

// Any even head_dim (up to 1024, for the shared memory): a warp per head, the normalised row in it.
constexpr int kQkWarps = 4;

template <class T>
__global__ void __launch_bounds__(kQkWarps * 32) qk_norm_rope_any_kernel(QkNormRopeParams p) {
  extern __shared__ float s_rows[];
  after_previous();
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

struct QkLaunch {
  QkNormRopeParams p;
  int vec_in, vec_out, vec_turn, sm_count;
  cudaStream_t st;
};

template <class T, int E, int LPH, int MODE, bool EXACT>
cudaError_t qk_launch_vec(const QkLaunch& a) {
  auto blocks = [&](int hb) {
    const int parts = (a.p.heads[0] + hb - 1) / hb + (a.p.heads[1] + hb - 1) / hb;
    return (unsigned)(((long long)a.p.tokens * parts * LPH + 255) / 256);
  };
  // one head a group until every SM has its 2048 threads twice over
  if (blocks(4) < 16ll * a.sm_count)
    return launch(qk_norm_rope_kernel<T, E, LPH, 1, MODE, EXACT>, dim3(blocks(1)), 256, 0, a.st, a.p, a.vec_in, a.vec_out,
                  a.vec_turn);
  return launch(qk_norm_rope_kernel<T, E, LPH, 4, MODE, EXACT>, dim3(blocks(4)), 256, 0, a.st, a.p, a.vec_in, a.vec_out,
                a.vec_turn);
}

template <class T, int E, int LPH>
cudaError_t qk_launch_mode(const QkLaunch& a, int mode) {
  const bool exact = a.p.head_dim == E * LPH;
  if (mode == kHalves) return exact ? qk_launch_vec<T, E, LPH, kHalves, true>(a) : qk_launch_vec<T, E, LPH, kHalves, false>(a);
  if (mode == kPairs) return exact ? qk_launch_vec<T, E, LPH, kPairs, true>(a) : qk_launch_vec<T, E, LPH, kPairs, false>(a);
  return exact ? qk_launch_vec<T, E, LPH, kPart, true>(a) : qk_launch_vec<T, E, LPH, kPart, false>(a);
}

template <class T>
cudaError_t qk_launch(const QkNormRopeParams& p, int sm_count, cudaStream_t st) {
  constexpr int S = (int)sizeof(T), E = 16 / S;  // 16 bytes a lane
  uintptr_t in = 0, out = 0;
  for (int i = 0; i < 2; ++i) {
    if (p.heads[i] == 0) continue;
    in |= reinterpret_cast<uintptr_t>(p.x[i]) | (uintptr_t)(p.in_stride[i] * S);
    out |= reinterpret_cast<uintptr_t>(p.out[i]) | (uintptr_t)(p.out_stride[i] * S);
  }
  const uintptr_t heads = (uintptr_t)(p.head_dim * S);  // heads lie one after the other
  in |= heads;
  out |= heads;
  QkLaunch a{p, in % 32 == 0 ? 2 : in % 16 == 0, out % 32 == 0 ? 2 : out % 16 == 0,
             (reinterpret_cast<uintptr_t>(p.cos_cache) | reinterpret_cast<uintptr_t>(p.sin_cache)) % 8 == 0 &&
                 p.rot_dim / 2 % 2 == 0,
             sm_count, st};
  const int half = p.rot_dim / 2, e = p.head_dim > 32 * E ? 8 : E;  // values of a lane
  const int mode = p.interleaved ? kPairs : p.rot_dim == p.head_dim ? kHalves : kPart;
  if (p.head_dim % e == 0 && p.head_dim <= 32 * e && (mode != kPart || half % e == 0)) {
    const int lanes = p.head_dim / e;
    if (e != E) return qk_launch_mode<T, 8, 32>(a, mode);
    if (lanes <= 8) return qk_launch_mode<T, E, 8>(a, mode);
    if (lanes <= 16) return qk_launch_mode<T, E, 16>(a, mode);
    return qk_launch_mode<T, E, 32>(a, mode);
  }
  const long long units = (long long)p.tokens * (p.heads[0] + p.heads[1]);
  return launch(qk_norm_rope_any_kernel<T>, dim3((unsigned)((units + kQkWarps - 1) / kQkWarps)), kQkWarps * 32,
                kQkWarps * p.head_dim * sizeof(float), st, p);
}

// ---- quantised writes and reads ------------------------------------------------------------------
//
// A group of G values: offset m = f16(min), scale s = f16((max - min) / 15), codes
// clamp(rint((x - m) / s), 0, 15) with the true quotient rounded to the nearest, ties to even.  The
// quotient is taken as (x - m) * (1 / s) in f32: three roundings, off by at most 3 * 2^-24 * 15.01 <
// 3e-6; a thread that holds one within 8e-6 of a tie settles its 8 codes in 64 bits.  (IEEE divisions
// instead of the product: 43 us for 8192 tokens of 8 heads of 128 in f32.)  8 values a lane: one
// 16-byte load (f16, bf16) or two (f32), one 32-bit store of codes; a group is 8 or 16 lanes.  A
// group of lanes takes HB heads of a token's keys or values, their loads in flight at once: bound
// by HBM.
constexpr int kKv4Lane = 8;

// A CTA's threads are rows of consecutive tokens; blockIdx.y names the heads, of keys or of values.
struct Kv4Lane {
  int l, head, which, token;  // lane of the row, first head, 0 keys 1 values
};
template <int HB>
__device__ __forceinline__ Kv4Lane kv4_lane(const Kv4View& c) {
  const int log_lanes = c.head_dim == 64 ? 3 : c.head_dim == 128 ? 4 : 5;
  const int which = blockIdx.y & 1, head = (int)(blockIdx.y >> 1) * HB;
  return {(int)threadIdx.x & ((1 << log_lanes) - 1), head, which,
          (int)(blockIdx.x << (8 - log_lanes)) + (int)(threadIdx.x >> log_lanes)};
}

// The lesser and the greater; NaN if one is.
__device__ __forceinline__ float min_nan(float a, float b) {
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

template <class T, int HB>
__global__ void __launch_bounds__(256) kv4_append_kernel(Kv4View c, const T* k, const T* v, const int* slots,
                                                         int tokens, long long k_stride, long long v_stride, int vec) {
  after_previous();
  const Kv4Lane at = kv4_lane<HB>(c);
  const int slot = at.token < tokens ? slots[at.token] : -1;
  const long long row0 = kv4_slot_row(c, slot, at.head);
  const bool on = row0 >= 0;
  const T* src = (at.which ? v + at.token * v_stride : k + at.token * k_stride) + at.head * c.head_dim + at.l * kKv4Lane;
  uint8_t* codes = at.which ? c.v_codes : c.k_codes;
  uint32_t* scales = at.which ? c.v_scales : c.k_scales;
  float x[HB][kKv4Lane];
#pragma unroll
  for (int i = 0; i < HB; ++i) {
#pragma unroll
    for (int e = 0; e < kKv4Lane; ++e) x[i][e] = 0.f;
    if (on && at.head + i < c.kv_heads)
      load_f32<T, kKv4Lane>(src + i * c.head_dim, vec, x[i]);
  }
  const int log_group = c.group == 64 ? 3 : 4;  // lanes of a group
  const int log_row = c.head_dim == 64 ? 3 : c.head_dim == 128 ? 4 : 5;
#pragma unroll
  for (int i = 0; i < HB; ++i) {
    float lo = x[i][0], hi = x[i][0];
#pragma unroll
    for (int e = 1; e < kKv4Lane; ++e) {
      lo = min_nan(lo, x[i][e]);
      hi = max_nan(hi, x[i][e]);
    }
    for (int off = 1 << (log_group - 1); off > 0; off >>= 1) {
      lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, off));
      hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, off));
    }
    if (!on || at.head + i >= c.kv_heads) continue;
    const float odd = lo * 0.f + hi * 0.f;  // NaN when a value is not finite, else 0
    // (max - min) / 15 rounded to f16, finite values past it saturating: in f32 when 2^-21 on either
    // side round alike (two roundings of 2^-24), else in 64 bits
    const float range = (hi - lo) * (1.f / 15.f);
    __half hs = __float2half_rn(fminf(range * (1.f + 4.8e-7f), 65504.f) + odd);
    if (__half_as_ushort(hs) != __half_as_ushort(__float2half_rn(fminf(range * (1.f - 4.8e-7f), 65504.f) + odd)))
      hs = __float2half_rn(fminf((float)(((double)hi - (double)lo) / 15.0), 65504.f) + odd);
    const __half hm = __float2half_rn(fminf(fmaxf(lo, -65504.f), 65504.f) + odd);
    const float s = __half2float(hs), m = __half2float(hm);
    uint32_t word = 0;
    if (s > 0.f) {
      const float inv = __frcp_rn(s);
      constexpr float kMagic = 12582912.f;  // 1.5 * 2^23: an integer in the low bits of a sum with it
      float off_tie = 0.f;
#pragma unroll
      for (int e = kKv4Lane - 1; e >= 0; --e) {
        const float d = x[i][e] - m;
        const float t = fmaf(d, inv, kMagic);
        off_tie = fmaxf(off_tie, fabsf(fmaf(d, inv, kMagic - t)));
        word = word * 16u + (__float_as_uint(t) - 0x4B400000u);  // 16 * word + code
      }
      // near a tie, or a group whose rounded offset or scale leaves its ends past 0 .. 15
      if (off_tie > 0.5f - 8e-6f || !((lo - m) * inv > -0.499f && (hi - m) * inv < 15.499f)) {
        word = 0;
#pragma unroll 1
        for (int e = kKv4Lane - 1; e >= 0; --e) {
          float xe = x[i][0];
#pragma unroll
          for (int q = 1; q < kKv4Lane; ++q)
            if (q == e) xe = x[i][q];
          word = word * 16u + (uint32_t)fmin(fmax(rint(((double)xe - (double)m) / (double)s), 0.0), 15.0);
        }
      }
    }
    const long long row = row0 + ((long long)i << c.shift);
    reinterpret_cast<uint32_t*>(codes)[(row << log_row) + at.l] = word;
    if ((at.l & ((1 << log_group) - 1)) == 0)
      scales[(row << (log_row - log_group)) + (at.l >> log_group)] =
          (uint32_t)__half_as_ushort(hs) | (uint32_t)__half_as_ushort(hm) << 16;
  }
}

template <class T, int HB>
__global__ void __launch_bounds__(256) kv4_gather_kernel(Kv4View c, T* k, T* v, const int* slots, int tokens,
                                                         long long k_stride, long long v_stride, int vec) {
  after_previous();
  const Kv4Lane at = kv4_lane<HB>(c);
  if (at.token >= tokens) return;
  const long long row0 = kv4_slot_row(c, slots[at.token], at.head);
  if (row0 < 0) return;
  const uint8_t* codes = at.which ? c.v_codes : c.k_codes;
  const uint32_t* scales = at.which ? c.v_scales : c.k_scales;
  T* dst = (at.which ? v + at.token * v_stride : k + at.token * k_stride) + at.head * c.head_dim + at.l * kKv4Lane;
  const int log_group = c.group == 64 ? 3 : 4, log_row = c.head_dim == 64 ? 3 : c.head_dim == 128 ? 4 : 5;
  uint32_t word[HB], pair[HB];
#pragma unroll
  for (int i = 0; i < HB; ++i) {
    const long long row = row0 + ((long long)(min(at.head + i, c.kv_heads - 1) - at.head) << c.shift);
    word[i] = reinterpret_cast<const uint32_t*>(codes)[(row << log_row) + at.l];
    pair[i] = scales[(row << (log_row - log_group)) + (at.l >> log_group)];
  }
#pragma unroll
  for (int i = 0; i < HB; ++i) {
    if (at.head + i >= c.kv_heads) break;
    const float s = __half2float(__ushort_as_half((unsigned short)pair[i]));
    const float m = __half2float(__ushort_as_half((unsigned short)(pair[i] >> 16)));
    float x[kKv4Lane];
#pragma unroll
    for (int e = 0; e < kKv4Lane; ++e) {
      // the nibble in the low bits of 1.5 * 2^23, read as f32: faster than a conversion
      const float code = __uint_as_float((word[i] >> (4 * e) & 15u) | 0x4B400000u) - 12582912.f;
      x[e] = fmaf(code, s, m);
    }
    store_f32<T, kKv4Lane>(dst + i * c.head_dim, vec, x);
  }
}

// 2: all rows on 32-byte boundaries, 1: on 16-byte boundaries.
template <class T>
int rows_vec(const void* k, const void* v, long long k_stride, long long v_stride) {
  const uintptr_t bits = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
                         (uintptr_t)(k_stride * (long long)sizeof(T)) | (uintptr_t)(v_stride * (long long)sizeof(T));
  return bits % 32 == 0 ? 2 : bits % 16 == 0 ? 1 : 0;
}

// Grid of HB heads a group: rows of 256 threads, (heads, keys and values).
dim3 kv4_grid(const Kv4View& c, int tokens, int hb) {
  const int rows = 256 / (c.head_dim / kKv4Lane);
  return dim3((unsigned)((tokens + (long long)rows - 1) / rows), 2u * (unsigned)((c.kv_heads + hb - 1) / hb));
}
// one head a group until every SM has its 2048 threads
constexpr int kKv4Heads = 4;
bool kv4_batched(const Kv4View& c, int tokens, int sm_count) {
  const dim3 g = kv4_grid(c, tokens, kKv4Heads);
  return (long long)g.x * g.y >= 8ll * sm_count;
}

template <class T>
cudaError_t append(const Kv4View& c, const void* k, const void* v, const int* slots, int tokens,
                   long long k_stride, long long v_stride, int sm_count, cudaStream_t st) {
  const int vec = rows_vec<T>(k, v, k_stride, v_stride);
  const T *kt = static_cast<const T*>(k), *vt = static_cast<const T*>(v);
  if (kv4_batched(c, tokens, sm_count))
    return launch(kv4_append_kernel<T, kKv4Heads>, kv4_grid(c, tokens, kKv4Heads), 256, 0, st, c, kt, vt, slots,
                  tokens, k_stride, v_stride, vec);
  return launch(kv4_append_kernel<T, 1>, kv4_grid(c, tokens, 1), 256, 0, st, c, kt, vt, slots, tokens, k_stride,
                v_stride, vec);
}

template <class T>
cudaError_t gather(const Kv4View& c, void* k, void* v, const int* slots, int tokens, long long k_stride,
                   long long v_stride, int sm_count, cudaStream_t st) {
  const int vec = rows_vec<T>(k, v, k_stride, v_stride);
  T *kt = static_cast<T*>(k), *vt = static_cast<T*>(v);
  if (kv4_batched(c, tokens, sm_count))
    return launch(kv4_gather_kernel<T, kKv4Heads>, kv4_grid(c, tokens, kKv4Heads), 256, 0, st, c, kt, vt, slots,
                  tokens, k_stride, v_stride, vec);
  return launch(kv4_gather_kernel<T, 1>, kv4_grid(c, tokens, 1), 256, 0, st, c, kt, vt, slots, tokens, k_stride,
                v_stride, vec);
}

}  // namespace

cudaError_t launch_paged_slots(const SlotsParams& p, int sm_count, cudaStream_t st) {
  // a token a thread while that fills the SMs at most once
  const bool few = p.max_tokens <= (long long)kSlotsThreads * sm_count;
  const long long per = kSlotsThreads * (few ? 1 : 4);
  const long long ctas = std::min((p.max_tokens + per - 1) / per, (long long)sm_count * 4);
  return launch(few ? paged_slots_kernel<1> : paged_slots_kernel<4>, dim3((unsigned)(ctas > 1 ? ctas + 1 : 1)), kSlotsThreads, 0, st, p);
}

cudaError_t launch_qk_norm_rope(const QkNormRopeParams& p, int dtype, int sm_count, cudaStream_t st) {
  switch (dtype) {
    case kTypeF32: return qk_launch<float>(p, sm_count, st);
    case kTypeF16: return qk_launch<__half>(p, sm_count, st);
    default: return qk_launch<__nv_bfloat16>(p, sm_count, st);
  }
}

cudaError_t launch_kv4_append(const Kv4View& c, const void* k, const void* v, const int* slots, int tokens,
                              long long k_stride, long long v_stride, int dtype, int sm_count, cudaStream_t st) {
  switch (dtype) {
    case kTypeF32: return append<float>(c, k, v, slots, tokens, k_stride, v_stride, sm_count, st);
    case kTypeF16: return append<__half>(c, k, v, slots, tokens, k_stride, v_stride, sm_count, st);
    default: return append<__nv_bfloat16>(c, k, v, slots, tokens, k_stride, v_stride, sm_count, st);
  }
}

cudaError_t launch_kv4_gather(const Kv4View& c, void* k, void* v, const int* slots, int tokens,
                              long long k_stride, long long v_stride, int dtype, int sm_count, cudaStream_t st) {
  switch (dtype) {
    case kTypeF32: return gather<float>(c, k, v, slots, tokens, k_stride, v_stride, sm_count, st);
    case kTypeF16: return gather<__half>(c, k, v, slots, tokens, k_stride, v_stride, sm_count, st);
    default: return gather<__nv_bfloat16>(c, k, v, slots, tokens, k_stride, v_stride, sm_count, st);
  }
}

}  // namespace tk
