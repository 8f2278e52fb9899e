// tk_kv4_attention.cuh -- what the kernels of attention over the 4-bit cache share: the work's
// partition, the joining of partial sums, conversions.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "tk_kv4.h"

namespace tk {
namespace {

constexpr int kStep = 128;  // tokens of a step
// Steps that a tile costs beside its own: queries, first loads, join (48 sequences of 64 to 8192: 65.9 us
// with 1, 62.7 with 2, 61.2 with 3; 32 of 512: 15.4, 15.7, 17.8.  Prompts: 2 x 256 tokens over 1500 to
// 4000 positions 111, 109, 116; 2048 tokens over themselves 139, 132, 132; 512 of them 33.1, 34.1, 39.1).
constexpr int kTileCost = 2;

// Work is (sequence, key head, row tile, step of 128 tokens) in this order, cut into equal runs, one
// per CTA; a tile counts kTileCost steps more than it has, before its first.  So long and short
// sequences, few and many, load the SMs alike, whatever the lengths, which only the device knows.  A
// run that ends inside a tile leaves its sums in the workspace; the CTA in whose run the tile begins
// describes it, and a second kernel joins the parts in the order of the CTAs.  A CTA has at most two
// parts: the end of a tile in slot 0, the beginning of one in slot 1.
struct Part {
  int token, rows, head, count;  // of the tile: the sequence's first query token, rows, key head; its parts (0: none)
  int row0, slot, pad0, pad1;    // the tile's first row; the slot of the first part
};

__device__ __forceinline__ float load_any(const void* base, long long i, int dtype) {
  if (dtype == kTypeF32) return static_cast<const float*>(base)[i];
  if (dtype == kTypeF16) return __half2float(static_cast<const __half*>(base)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(base)[i]);
}
// 8 consecutive values of a row.
__device__ __forceinline__ void load_row8(const void* base, long long i, int dtype, float (&v)[8]) {
  const int size = dtype == kTypeF32 ? 4 : 2;
  const uint8_t* src = static_cast<const uint8_t*>(base) + i * size;
  if (reinterpret_cast<uintptr_t>(src) & 15) {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = load_any(base, i + k, dtype);
    return;
  }
  const uint4 x = reinterpret_cast<const uint4*>(src)[0];
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  if (dtype == kTypeF32) {
    const uint4 z = reinterpret_cast<const uint4*>(src)[1];
    const uint32_t w2[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = __uint_as_float(w[k]), v[4 + k] = __uint_as_float(w2[k]);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[2 * k] = dtype == kTypeF16 ? __half2float(__ushort_as_half((unsigned short)w[k])) : __uint_as_float(w[k] << 16);
      v[2 * k + 1] = dtype == kTypeF16 ? __half2float(__ushort_as_half((unsigned short)(w[k] >> 16)))
                                       : __uint_as_float(w[k] & 0xFFFF0000u);
    }
  }
}
__device__ __forceinline__ void store_any(void* base, long long i, int dtype, float v) {
  if (dtype == kTypeF32)
    static_cast<float*>(base)[i] = v;
  else if (dtype == kTypeF16)
    static_cast<__half*>(base)[i] = __float2half_rn(v);
  else
    static_cast<__nv_bfloat16*>(base)[i] = __float2bfloat16_rn(v);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float half_lo(uint32_t w) { return __half2float(__ushort_as_half((unsigned short)w)); }
__device__ __forceinline__ float half_hi(uint32_t w) {
  return __half2float(__ushort_as_half((unsigned short)(w >> 16)));
}
// Two f32 as f16 (a in the low half), and what that leaves of them.
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  uint32_t y;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(b), "f"(a));
  return y;
}
__device__ __forceinline__ void split_f16(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = pack_f16(a, b);
  lo = pack_f16(a - half_lo(hi), b - half_hi(hi));
}

// kept = kept * g + x, or x where nothing is kept yet.  Returns what its rounding drops, so that a long row of
// such sums is off by no more than a short one (compensated summation).
__device__ __forceinline__ float keep(bool any, float& kept, float g, float x) {
  if (!any) {  // (g may be anything)
    kept = x;
    return 0.f;
  }
  const float sum = fmaf(kept, g, x), drop = x + fmaf(kept, g, -sum);
  kept = sum;
  return drop;
}

struct Sequence {
  int first, n;     // query tokens
  int kv;           // visible positions, at most the table's reach
  int last;         // kv_len - n: query i sees the positions below last + i + 1
  int tiles;        // row tiles
  int steps;        // of a tile that sees all of it, its cost among them
};
// Tiles of many rows count the steps that their own rows see (32 + 8 heads of 128, 2048 tokens over
// themselves: 132 us instead of 194, 8192: 1.43 ms instead of 2.55), smaller ones all of the sequence's.
constexpr int kManyRows = 128;
__device__ __forceinline__ PromptTiles prompt_of(const Sequence& s, int per) {
  return prompt_tiles(s.tiles, per, kTileCost, s.last, s.kv);
}
template <int ROWS>
__device__ __forceinline__ long long work_of(const Sequence& s, int per) {  // of a key head
  if constexpr (ROWS == kManyRows) return prompt_work(prompt_of(s, per));
  return (long long)s.steps * s.tiles;
}
template <int ROWS>
__device__ __forceinline__ Sequence sequence(const Kv4AttentionParams& p, int b, int per) {
  Sequence s;
  if (p.query_start) {
    s.first = min(max(p.query_start[b], 0), p.tokens);
    s.n = max(min(p.query_start[b + 1], p.tokens) - s.first, 0);
  } else {
    s.first = b;
    s.n = 1;
  }
  const int len = max(p.kv_lens[b], 0);
  s.last = len - s.n;
  s.kv = (int)min((long long)len, (long long)p.max_blocks << p.cache.shift);
  s.tiles = (int)(((long long)s.n * per + ROWS - 1) / ROWS);
  s.steps = kTileCost + (s.kv + kStep - 1) / kStep;  // kv < 2^31 - 1024
  return s;
}

// The part of a tile that a run holds.
struct Tile {
  int b, head, rt;  // sequence, key head, row tile
  int steps;        // of the tile, its cost among them
  int c0, c1;       // those of the run
  Sequence s;
};

// A CTA's run, and its length in general.
struct Run {
  long long length, start, stop;
};
// Finds it and its first tile, and marks that no tile begins in it yet.  False: nothing to do.
template <int ROWS, int THREADS>
__device__ __forceinline__ bool find_run(const Kv4AttentionParams& p, int per, Part* parts, Run& r, Tile& cur) {
  constexpr int W = THREADS / 32;
  __shared__ long long s_warp[W];
  __shared__ long long s_at;
  __shared__ int s_seq;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, hk = p.cache.kv_heads;
  const int chunk = (p.batch + THREADS - 1) / THREADS;
  const int b0 = (int)min((long long)p.batch, (long long)tid * chunk), b1 = min(p.batch, b0 + chunk);
  long long mine = 0;
  for (int b = b0; b < b1; ++b) {
    const Sequence s = sequence<ROWS>(p, b, per);
    mine += work_of<ROWS>(s, per) * hk;
  }
  long long inc = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const long long o = __shfl_up_sync(0xffffffffu, inc, off);
    if (lane >= off) inc += o;
  }
  if (lane == 31) s_warp[warp] = inc;
  __syncthreads();
  long long before = inc - mine, total = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    if (w < warp) before += s_warp[w];
    total += s_warp[w];
  }
  // (a quotient in f64, rounded up at least: 64-bit division takes as long as a load)
  const long long run = (long long)__dmul_ru((double)total, p.inv_ctas) + 1;
  const long long start = run * blockIdx.x, stop = min(start + run, total);
  if (tid == 0) parts[blockIdx.x].count = 0;
  if (start >= stop) return false;
  if (start >= before && start < before + mine) {  // one thread's
    long long at = before;
    int b = b0;
    for (;; ++b) {
      const Sequence s = sequence<ROWS>(p, b, per);
      const long long w = work_of<ROWS>(s, per) * hk;
      if (start < at + w) break;
      at += w;
    }
    s_seq = b;
    s_at = start - at;
  }
  __syncthreads();
  cur.b = s_seq;
  cur.s = sequence<ROWS>(p, cur.b, per);
  // which head, or head and tile, by a quotient in f64, off by one at most
  const long long of_unit = ROWS == kManyRows ? work_of<ROWS>(cur.s, per) : cur.s.steps;
  long long unit = (long long)((double)s_at / (double)of_unit);
  if (unit * of_unit > s_at) --unit;
  if ((unit + 1) * of_unit <= s_at) ++unit;
  const long long rest = s_at - unit * of_unit;
  if constexpr (ROWS == kManyRows) {
    const PromptTiles t = prompt_of(cur.s, per);
    cur.head = (int)unit;
    cur.rt = prompt_find(t, rest, &cur.c0);
    cur.steps = prompt_steps(t, cur.rt);
  } else {
    cur.head = (int)unit / cur.s.tiles;
    cur.rt = (int)unit - cur.head * cur.s.tiles;
    cur.c0 = (int)rest;
    cur.steps = cur.s.steps;
  }
  cur.c1 = (int)min((long long)cur.steps, cur.c0 + (stop - start));
  r = Run{run, start, stop};
  return true;
}

// The tile after cur within the run: the next rows, head, sequence.  at: its first step, below stop.
template <int ROWS>
__device__ __forceinline__ void next_tile(const Kv4AttentionParams& p, int per, long long at, long long stop, Tile& cur) {
  cur.c0 = 0;
  if (++cur.rt == cur.s.tiles) {
    cur.rt = 0;
    if (++cur.head == p.cache.kv_heads) {
      cur.head = 0;
      do {
        cur.s = sequence<ROWS>(p, ++cur.b, per);
      } while (cur.s.tiles == 0);
    }
  }
  cur.steps = ROWS == kManyRows ? prompt_steps(prompt_of(cur.s, per), cur.rt) : cur.s.steps;
  cur.c1 = (int)min((long long)cur.steps, stop - at);
}

// Joins the parts of the tile that begins in the run of CTA blockIdx.x, RC of its rows.  W warps a row,
// each with every W-th part, then in the order of the warps.
template <int D, int ROWS, int RC, int W>
__global__ void __launch_bounds__(RC * W * 32) kv4_join_kernel(Kv4AttentionParams p, int dtype) {
  __shared__ float s_num[RC][W][2];
  __shared__ float s_v[RC][W][D];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const Part* parts = static_cast<const Part*>(p.workspace);
  const float* sums = reinterpret_cast<const float*>(parts + gridDim.x);
  constexpr int kSlot = ROWS * (D + 2);
  const Part part = parts[blockIdx.x];
  if (part.count == 0) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r0 = warp / W, w = warp % W;
  const int row = blockIdx.y * RC + r0;
  constexpr int V = D == 64 ? 2 : 4, E = D / (32 * V);  // values of a load, loads of a row
  constexpr int U = 8 / E;                              // parts in flight
  float top = -INFINITY, sum = 0.f, v[E][V];
#pragma unroll
  for (int e = 0; e < E; ++e)
#pragma unroll
    for (int k = 0; k < V; ++k) v[e][k] = 0.f;
  for (int i0 = w; i0 < part.count; i0 += W * U) {
    float2 num[U];
    float x[U][E][V];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = min(i0 + u * W, part.count - 1);  // one that counts, read again
      const float* s = sums + ((size_t)(blockIdx.x + i) * 2 + (i == 0 ? part.slot : 0)) * kSlot;
      num[u] = *reinterpret_cast<const float2*>(s + ROWS * D + 2 * row);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float* src = s + row * D + (e * 32 + lane) * V;
        if constexpr (V == 4)
          *reinterpret_cast<float4*>(x[u][e]) = *reinterpret_cast<const float4*>(src);
        else
          *reinterpret_cast<float2*>(x[u][e]) = *reinterpret_cast<const float2*>(src);
      }
    }
    float now = top;
#pragma unroll
    for (int u = 0; u < U; ++u) now = fmaxf(now, num[u].x);
    const float f0 = top == -INFINITY ? 1.f : ex2(top - now);  // no reference: sums of 0, or of NaN
    top = now;
    sum *= f0;
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
      for (int k = 0; k < V; ++k) v[e][k] *= f0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i0 + u * W >= part.count) break;
      const float f = num[u].x == -INFINITY ? 1.f : ex2(num[u].x - top);
      sum = fmaf(num[u].y, f, sum);
#pragma unroll
      for (int e = 0; e < E; ++e)
#pragma unroll
        for (int k = 0; k < V; ++k) v[e][k] = fmaf(x[u][e][k], f, v[e][k]);
    }
  }
  if (lane == 0) {
    s_num[r0][w][0] = top;
    s_num[r0][w][1] = sum;
  }
#pragma unroll
  for (int e = 0; e < E; ++e)
#pragma unroll
    for (int k = 0; k < V; ++k) s_v[r0][w][(e * 32 + lane) * V + k] = v[e][k];
  __syncthreads();
  if (row >= part.rows) return;
  float f[W];
  top = -INFINITY;
  sum = 0.f;
#pragma unroll
  for (int i = 0; i < W; ++i) top = fmaxf(top, s_num[r0][i][0]);
#pragma unroll
  for (int i = 0; i < W; ++i) {
    f[i] = s_num[r0][i][0] == -INFINITY ? 1.f : ex2(s_num[r0][i][0] - top);
    sum = fmaf(s_num[r0][i][1], f[i], sum);
  }
  const int per = p.q_heads / p.cache.kv_heads, q = part.row0 + row;
  const long long at = (long long)(part.token + q / per) * p.o_stride + (long long)(part.head * per + q % per) * D;
  for (int d = w * 32 + lane; d < D; d += W * 32) {
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) x = fmaf(s_v[r0][i][d], f[i], x);
    store_any(p.o, at + d, dtype, sum == 0.f ? 0.f : x / sum);
  }
}

// Bytes for the partial sums of CTAs with tiles of `rows` rows.
inline size_t attention_workspace(int ctas, int rows, int head_dim) {
  return (size_t)ctas * (sizeof(Part) + 2 * (size_t)rows * (head_dim + 2) * sizeof(float));
}

}  // namespace

// tk_kv4_prompt.cu
bool kv4_prompt_takes(const Kv4AttentionParams& p, int dtype);
size_t kv4_prompt_workspace(int head_dim, int sm_count);
cudaError_t launch_kv4_prompt(Kv4AttentionParams p, int dtype, int sm_count, cudaStream_t st);

}  // namespace tk
