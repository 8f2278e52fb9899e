// tk_kv4_attention.cu -- attention over the key/value cache held in 4 bits.
//
// For query i of the n query tokens of a sequence with kv_len tokens in the cache (those n among
// them): o = sum_p w_p v_p, w = softmax_p(scale * q . k_p) over the positions p < kv_len - n + i + 1,
// with k, v = code * scale + offset.  A position whose page is not in the cache counts as absent; a
// query that sees no position gets zeros.
//
// The mathematics.  Scales and offsets stay out of the products (c: codes, per group of dimensions):
//     q . k   = sum_g s_k (q . c)_g + m_k (sum q)_g
//     sum p v = sum (p s_v) (c - 8)  +  sum p (m_v + 8 s_v)
// so both products are f16 x f16 tensor-core products with exact codes: keys as f16 subnormals
// (c * 2^-24, or c * 2^-20 from the high nibble, the matching queries divided by 16: one AND per two
// codes), values as c - 8 (without the shift the sums would carry 7.5 times the weights, and a long
// flat softmax would lose its digits against it).  f32 queries and weights are split into two f16
// (22 bits), which take the rows g and g + 8 of the same m16n8k16 product: the heads of a group and
// the query tokens of a sequence (rows, 8 to a tile) fill the upper half, the remainders the lower.
// mma.sync and not tcgen05: one token of a head group is 8 rows, an eighth of tcgen05's smallest
// tile, whose operands would also have to pass through shared memory unpacked.
//
// Softmax in base 2 with a running reference per row: w = 2^(s - r) s_v must fit f16, so r follows
// max(s + log2 s_v) and is moved (sums rescaled) only when a weight would leave [0, 2^15].
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cstdint>

#include "tk_kv4.h"

namespace tk {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kRows = 8;       // rows (query token, head of the group) of a tile
constexpr int kUnit = 16;      // tokens of a warp's step; a page holds whole units
constexpr int kStep = kUnit * kWarps;
constexpr int kStages = 4;

// Work is (sequence, key head, row tile, step of 64 tokens) in this order, cut into equal runs, one
// per CTA (Kv4Run).  A run that ends inside a (sequence, head, tile) leaves its sums in the
// workspace; the CTA in whose run the tile begins describes it, and a second kernel joins the parts
// in the order of the CTAs.  A CTA has at most two parts: the end of a tile in slot 0, the beginning
// of one in slot 1.
struct Part {
  int token, rows, head, count;  // first row's query token... of the tile; parts to join (0: none)
  int row0, slot, pad0, pad1;    // first row of the tile; the slot of the first part
};

size_t part_bytes(int head_dim) { return (size_t)kRows * (head_dim + 2) * sizeof(float); }

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

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
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
__device__ __forceinline__ uint32_t pack2(__half a, __half b) {
  return (uint32_t)__half_as_ushort(a) | (uint32_t)__half_as_ushort(b) << 16;
}
__device__ __forceinline__ float half_lo(uint32_t w) { return __half2float(__ushort_as_half((unsigned short)w)); }
__device__ __forceinline__ float half_hi(uint32_t w) {
  return __half2float(__ushort_as_half((unsigned short)(w >> 16)));
}
// Two codes less 8 from bits 0-3 (codes_lo) or 4-7 (codes_hi) of the halves of x: as 1024 + c or
// 1024 + 16 c by the bits of the exponent, then exact f16 arithmetic.
__device__ __forceinline__ uint32_t codes_lo(uint32_t x) {
  x = (x & 0x000F000Fu) | 0x64006400u;
  const uint32_t k = 0x64086408u;  // 1032
  uint32_t y;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(y) : "r"(x), "r"(k));
  return y;
}
__device__ __forceinline__ uint32_t codes_hi(uint32_t x) {
  x = (x & 0x00F000F0u) | 0x64006400u;
  const uint32_t f = 0x2C002C00u, k = 0xD480D480u;  // 1/16, -72
  uint32_t y;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(y) : "r"(x), "r"(f), "r"(k));
  return y;
}

// A stage of a warp's ring: 16 tokens of codes and pairs.  16-byte pieces are placed so that no two
// lanes of a load meet in a bank: the keys of token x in row krow(x), piece c ^ kflip(x); the values
// of token 4t + r in row 4r + t, piece c ^ vflip(t).
template <int D, int G>
struct Stage {
  static constexpr int NG = D / G;
  static constexpr int kRowBytes = D / 2;
  static constexpr int kPieces = D / 32;  // 16-byte pieces of a row
  static constexpr int kCodes = kUnit * kRowBytes;
  static constexpr int kPairs = kUnit * NG * 4;
  static constexpr int kBytes = 2 * (kCodes + kPairs);
  static __device__ __forceinline__ int krow(int x) { return D == 64 ? x ^ ((x >> 2 & 1) << 1) : x; }
  static __device__ __forceinline__ int kflip(int x) {
    if (D == 64) return 0;
    if (D == 128) return (x >> 2 & 1) << 1;
    return G == 128 ? (x & 1) << 2 : (x & 1) << 1 | (x >> 2 & 1) << 2;
  }
  static __device__ __forceinline__ int vflip(int t) { return D == 64 ? 0 : D == 128 ? (t >> 1) << 1 : t << 1; }
  static __device__ __forceinline__ int key_at(int token, int byte) {
    return krow(token) * kRowBytes + ((byte / 16 ^ kflip(token)) * 16 + byte % 16);
  }
  static __device__ __forceinline__ int value_at(int token, int byte) {
    return ((token & 3) * 4 + token / 4) * kRowBytes + ((byte / 16 ^ vflip(token / 4)) * 16 + byte % 16);
  }
};

struct Sequence {
  int first, n;     // query tokens
  int kv;           // visible positions, at most the table's reach
  int last;         // kv_len - n: query i sees the positions below last + i + 1
  int tiles;        // row tiles
  int steps;        // of a tile; 1 at least, so that empty contexts get their zeros
};
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
  s.tiles = (int)(((long long)s.n * per + kRows - 1) / kRows);
  s.steps = max(1, (s.kv + kStep - 1) / kStep);  // kv < 2^31 - 1024
  return s;
}

template <int D, int G>
__global__ void __launch_bounds__(kThreads, D == 256 ? 2 : 3) kv4_attention_kernel(Kv4AttentionParams p, int dtype) {
  using S = Stage<D, G>;
  constexpr int NG = S::NG, KS = D / 16, NT = D / 8;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ long long s_warp[kWarps];
  __shared__ long long s_at;
  __shared__ int s_seq;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int per = p.q_heads / p.cache.kv_heads, hk = p.cache.kv_heads;
  Part* parts = static_cast<Part*>(p.workspace);
  float* sums = reinterpret_cast<float*>(parts + gridDim.x);
  constexpr int kSlot = kRows * (D + 2);

  // ---- this CTA's run ----
  const int chunk = (p.batch + kThreads - 1) / kThreads;
  const int b0 = (int)min((long long)p.batch, (long long)tid * chunk), b1 = min(p.batch, b0 + chunk);
  long long mine = 0;
  for (int b = b0; b < b1; ++b) {
    const Sequence s = sequence(p, b, per);
    mine += (long long)s.steps * s.tiles * hk;
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
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += s_warp[w];
    total += s_warp[w];
  }
  const long long run = (total + gridDim.x - 1) / gridDim.x;
  const long long start = run * blockIdx.x, stop = min(start + run, total);
  if (tid == 0) parts[blockIdx.x].count = 0;
  if (start >= stop) return;
  if (start >= before && start < before + mine) {  // one thread's
    long long at = before;
    int b = b0;
    for (;; ++b) {
      const Sequence s = sequence(p, b, per);
      const long long w = (long long)s.steps * s.tiles * hk;
      if (start < at + w) break;
      at += w;
    }
    s_seq = b;
    s_at = start - at;
  }
  __syncthreads();
  int b = s_seq;
  long long offset = s_at;  // of the run's next step in its sequence

  uint8_t* ring = smem + warp * kStages * S::kBytes;
  const uint32_t ring_addr = (uint32_t)__cvta_generic_to_shared(ring);
  float* joint = reinterpret_cast<float*>(ring);  // after the ring: 8 rows of D sums, 8 x (reference, l)

  for (long long at = start; at < stop; ++b, offset = 0) {
    const Sequence s = sequence(p, b, per);
    const long long in_seq = (long long)s.steps * s.tiles * hk;
    while (at < stop && offset < in_seq) {
      const int unit = (int)(offset / s.steps), s0 = (int)(offset % s.steps);
      const int s1 = (int)min((long long)s.steps, s0 + (stop - at));
      const int head = unit / s.tiles, row0 = (unit % s.tiles) * kRows;
      const int rows = min(kRows, s.n * per - row0);
      const bool whole = s0 == 0 && s1 == s.steps;
      // positions that the tile's last row sees, and this lane's row
      const int see_tile = min(s.kv, s.last + (row0 + rows - 1) / per + 1);
      const int my_row = row0 + min(g, rows - 1);
      const int see = min(s.kv, s.last + my_row / per + 1);
      const int* table = p.block_tables + (size_t)b * p.max_blocks;

      // ---- queue of loads ----
      unsigned valid = 0;
      auto page_of = [&](int step) {
        const int pos = step * kStep + warp * kUnit;
        return step < s1 && pos < see_tile ? __ldg(table + (pos >> p.cache.shift)) : -1;
      };
      auto issue = [&](int stage, int step, int page) {
        const int pos = step * kStep + warp * kUnit;
        const long long row = kv4_row(p.cache, page, head, pos & ((1 << p.cache.shift) - 1));
        valid &= ~(1u << stage);
        if (row >= 0) {
          valid |= 1u << stage;
          const uint32_t dst = ring_addr + stage * S::kBytes;
          const uint8_t* kc = p.cache.k_codes + row * S::kRowBytes;
          const uint8_t* vc = p.cache.v_codes + row * S::kRowBytes;
#pragma unroll
          for (int i = 0; i < S::kCodes / 512; ++i) {
            const int piece = i * 32 + lane, token = piece / S::kPieces, byte = piece % S::kPieces * 16;
            cp_async16(dst + S::key_at(token, byte), kc + piece * 16);
            cp_async16(dst + S::kCodes + S::value_at(token, byte), vc + piece * 16);
          }
          if ((lane & 15) < 4 * NG) {
            const uint32_t* src = (lane < 16 ? p.cache.k_scales : p.cache.v_scales) + row * NG + (lane & 15) * 4;
            cp_async16(dst + 2 * S::kCodes + (lane < 16 ? 0 : S::kPairs) + (lane & 15) * 16, src);
          }
        }
        cp_commit();
      };
#pragma unroll
      for (int i = 0; i < kStages - 1; ++i) issue(i, s0 + i, page_of(s0 + i));
      int page_next = page_of(s0 + kStages - 1);

      // ---- queries: scaled, normalised by a power of two, split ----
      uint32_t qf[KS][4];
      float qsum[NG], unscale;
      {
        float q[D / 4];  // the lane's dimensions of row g: G/4 consecutive ones of each group
        const long long at_q = (long long)(s.first + my_row / per) * p.q_stride +
                               (long long)(head * per + my_row % per) * D;
        const float f = p.scale * 1.4426950408889634f;
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < D / 4; ++i) {
          const int d = i / (G / 4) * G + t * (G / 4) + i % (G / 4);
          q[i] = load_any(p.q, at_q + d, dtype) * f;
          top = fmaxf(top, fabsf(q[i]));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // the largest becomes 2^14 .. 2^15; a row of zeros, infinities or NaN goes as it is
        int e = 0;
        if (top > 0.f && top < INFINITY) e = min(max(14 - ilogbf(top), -100), 120);
        const float norm = ldexpf(1.f, e);
        unscale = ldexpf(1.f, 24 - e);
#pragma unroll
        for (int y = 0; y < NG; ++y) {
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < G / 4; ++i) sum += q[y * (G / 4) + i];
          sum += __shfl_xor_sync(0xffffffffu, sum, 1);
          sum += __shfl_xor_sync(0xffffffffu, sum, 2);
          qsum[y] = sum;
        }
#pragma unroll
        for (int w = 0; w < D / 32; ++w)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float x[4];  // codes 2h, 2h + 4 of the word, then 2h + 1, 2h + 5 (a factor 16 up)
            x[0] = q[8 * w + 2 * h] * norm;
            x[1] = q[8 * w + 2 * h + 4] * norm;
            x[2] = q[8 * w + 2 * h + 1] * norm * 0.0625f;
            x[3] = q[8 * w + 2 * h + 5] * norm * 0.0625f;
            __half hi[4], lo[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              hi[i] = __float2half_rn(x[i]);
              lo[i] = __float2half_rn(x[i] - __half2float(hi[i]));
            }
            uint32_t(&a)[4] = qf[2 * w + h];
            a[0] = pack2(hi[0], hi[1]);
            a[1] = pack2(lo[0], lo[1]);
            a[2] = pack2(hi[2], hi[3]);
            a[3] = pack2(lo[2], lo[3]);
          }
      }

      float o[NT][4], off_sum[NG], l = 0.f, ref = -INFINITY;  // weights are 2^(s - ref + 10) s_v
#pragma unroll
      for (int i = 0; i < NT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
#pragma unroll
      for (int y = 0; y < NG; ++y) off_sum[y] = 0.f;

      // ---- the steps ----
      for (int step = s0; step < s1; ++step) {
        const int stage = (step - s0) % kStages;
        cp_wait<kStages - 2>();
        __syncwarp();
        const bool there = valid >> stage & 1;
        issue((stage + kStages - 1) % kStages, step + kStages - 1, page_next);
        page_next = page_of(step + kStages);
        if (!there) continue;
        const uint8_t* st = ring + stage * S::kBytes;
        const uint32_t* kpair = reinterpret_cast<const uint32_t*>(st + 2 * S::kCodes) + 4 * t * NG;
        const uint32_t* vpair = reinterpret_cast<const uint32_t*>(st + 2 * S::kCodes + S::kPairs) + 4 * t * NG;
        const int left = see - (step * kStep + warp * kUnit + 4 * t);  // of the lane's 4 tokens, row g sees so many

        // scores of tokens 4t + r
        float sc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int y = 0; y < NG; ++y) {
          float c[2][4];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            c[j][0] = c[j][1] = c[j][2] = c[j][3] = 0.f;
            const int token = 4 * (g >> 1) + 2 * j + (g & 1);
            uint32_t w[G / 32];
            const uint8_t* src = st + S::key_at(token, y * (G / 2) + t * (G / 8));
            if constexpr (G == 128)
              *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(src);
            else
              *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(src);
#pragma unroll
            for (int i = 0; i < G / 32; ++i) {
              const int ks = y * (G / 16) + 2 * i;
              mma16816(c[j], qf[ks], w[i] & 0x000F000Fu, w[i] & 0x00F000F0u);
              const uint32_t v = w[i] >> 8;
              mma16816(c[j], qf[ks + 1], v & 0x000F000Fu, v & 0x00F000F0u);
            }
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const uint32_t pair = kpair[r * NG + y];
            const float dot = c[r >> 1][r & 1] + c[r >> 1][2 + (r & 1)];
            sc[r] += dot * unscale * half_lo(pair) + qsum[y] * half_hi(pair);
          }
        }

        // reference: the row's largest s + log2 of the value scale
        float vs[NG][4], vm[NG][4], top = -INFINITY;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float most = 5.9604645e-8f;  // 2^-24, the least f16
#pragma unroll
          for (int y = 0; y < NG; ++y) {
            const uint32_t pair = r < left ? vpair[r * NG + y] : 0u;
            vs[y][r] = half_lo(pair);
            vm[y][r] = fmaf(vs[y][r], 8.f, half_hi(pair));
            most = fmaxf(most, fabsf(vs[y][r]));
          }
          if (r >= left) sc[r] = -INFINITY;
          top = fmaxf(top, sc[r] + lg2(most));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const bool move = top > ref + 5.f;
        if (__any_sync(0xffffffffu, move)) {
          const float f = move ? ex2(ref - top) : 1.f;  // 0 at first
          if (move) ref = top;
          l *= f;
#pragma unroll
          for (int y = 0; y < NG; ++y) off_sum[y] *= f;
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            o[i][0] *= f;
            o[i][1] *= f;
            o[i][2] *= f;
            o[i][3] *= f;
          }
        }
        const float base = ref == -INFINITY ? 0.f : ref - 10.f;
        float pr[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          pr[r] = ex2(sc[r] - base);
          l += pr[r];
        }

#pragma unroll
        for (int y = 0; y < NG; ++y) {
          uint32_t a[4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float w0 = pr[2 * h] * vs[y][2 * h], w1 = pr[2 * h + 1] * vs[y][2 * h + 1];
            const __half h0 = __float2half_rn(w0), h1 = __float2half_rn(w1);
            a[2 * h] = pack2(h0, h1);
            a[2 * h + 1] = pack2(__float2half_rn(w0 - __half2float(h0)), __float2half_rn(w1 - __half2float(h1)));
            off_sum[y] = fmaf(pr[2 * h], vm[y][2 * h], fmaf(pr[2 * h + 1], vm[y][2 * h + 1], off_sum[y]));
          }
          uint32_t w[4][G / 64];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const uint8_t* src = st + S::kCodes + S::value_at(4 * t + r, y * (G / 2) + g * (G / 16));
            if constexpr (G == 128)
              *reinterpret_cast<uint2*>(w[r]) = *reinterpret_cast<const uint2*>(src);
            else
              w[r][0] = *reinterpret_cast<const uint32_t*>(src);
          }
#pragma unroll
          for (int v = 0; v < G / 64; ++v)
#pragma unroll
            for (int k = 0; k < 4; ++k) {  // byte k of the four tokens' words: dimensions 2k, 2k + 1
              const uint32_t x = __byte_perm(w[0][v], w[1][v], k | k << 4 | (k + 4) << 8 | (k + 4) << 12);
              const uint32_t z = __byte_perm(w[2][v], w[3][v], k | k << 4 | (k + 4) << 8 | (k + 4) << 12);
              const int n = (y * (G / 64) + v) * 8 + 2 * k;
              mma16816(o[n], a, codes_lo(x), codes_lo(z));
              mma16816(o[n + 1], a, codes_hi(x), codes_hi(z));
            }
        }
      }
      cp_wait<0>();
      __syncwarp();

      // ---- join the four warps ----
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
#pragma unroll
      for (int y = 0; y < NG; ++y) {
        off_sum[y] += __shfl_xor_sync(0xffffffffu, off_sum[y], 1);
        off_sum[y] += __shfl_xor_sync(0xffffffffu, off_sum[y], 2);
#pragma unroll
        for (int v = 0; v < G / 64; ++v)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int n = (y * (G / 64) + v) * 8 + e;
            const int d = y * G + 8 * v + e;  // of column 0; the next column is G/8 on
            joint[g * D + d + 2 * t * (G / 8)] = o[n][0] + o[n][2] + off_sum[y];
            joint[g * D + d + (2 * t + 1) * (G / 8)] = o[n][1] + o[n][3] + off_sum[y];
          }
      }
      if (t == 0) {
        joint[kRows * D + 2 * g] = ref;
        joint[kRows * D + 2 * g + 1] = l;
      }
      __syncthreads();
      constexpr int kJoint = kStages * S::kBytes / 4;  // floats from warp to warp
      const float* all = reinterpret_cast<const float*>(smem);
      const int slot = at == start ? 0 : 1;
      float* out = sums + ((size_t)blockIdx.x * 2 + slot) * kSlot;
      for (int i = tid; i < kRows * D; i += kThreads) {
        const int row = i / D, d = i % D;
        float top = -INFINITY, sum = 0.f, v = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, all[w * kJoint + kRows * D + 2 * row]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float r = all[w * kJoint + kRows * D + 2 * row];
          const float f = r == -INFINITY ? 0.f : ex2(r - top);
          const float lw = all[w * kJoint + kRows * D + 2 * row + 1];
          // a row of NaN scores never moves its reference: its sums are NaN
          sum += r == -INFINITY ? lw : lw * f;
          v += r == -INFINITY ? all[w * kJoint + i] : all[w * kJoint + i] * f;
        }
        if (whole) {
          if (row < rows) {
            const int q = row0 + row;
            store_any(p.o, (long long)(s.first + q / per) * p.o_stride + (long long)(head * per + q % per) * D + d,
                      dtype, sum == 0.f ? 0.f : v / sum);
          }
        } else {
          out[i] = v;
          if (d == 0) {
            out[kRows * D + 2 * row] = top;
            out[kRows * D + 2 * row + 1] = sum;
          }
        }
      }
      if (!whole && s0 == 0 && tid == 0) {  // the tile begins here: where its parts are
        const long long end = at + s.steps;
        parts[blockIdx.x] = Part{s.first, rows, head, (int)((end - 1) / run - blockIdx.x + 1), row0, slot, 0, 0};
      }
      __syncthreads();
      at += s1 - s0;
      offset += s1 - s0;
    }
  }
}

template <int D>
__global__ void __launch_bounds__(kRows * 32) kv4_join_kernel(Kv4AttentionParams p, int dtype) {
  const Part* parts = static_cast<const Part*>(p.workspace);
  const float* sums = reinterpret_cast<const float*>(parts + gridDim.x);
  constexpr int kSlot = kRows * (D + 2);
  const Part part = parts[blockIdx.x];
  const int row = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (row >= part.rows || part.count == 0) return;
  const int per = p.q_heads / p.cache.kv_heads;
  auto base = [&](int i) { return sums + ((size_t)(blockIdx.x + i) * 2 + (i == 0 ? part.slot : 0)) * kSlot; };
  float top = -INFINITY;
  for (int i = 0; i < part.count; ++i) top = fmaxf(top, base(i)[kRows * D + 2 * row]);
  float sum = 0.f, v[D / 32];
#pragma unroll
  for (int e = 0; e < D / 32; ++e) v[e] = 0.f;
  for (int i = 0; i < part.count; ++i) {
    const float* s = base(i);
    const float r = s[kRows * D + 2 * row];
    const float f = r == -INFINITY ? 1.f : ex2(r - top);  // no reference: sums of 0, or of NaN
    sum += s[kRows * D + 2 * row + 1] * f;
#pragma unroll
    for (int e = 0; e < D / 32; ++e) v[e] += s[row * D + e * 32 + lane] * f;
  }
  const int q = part.row0 + row;
  const long long at = (long long)(part.token + q / per) * p.o_stride + (long long)(part.head * per + q % per) * D;
#pragma unroll
  for (int e = 0; e < D / 32; ++e) store_any(p.o, at + e * 32 + lane, dtype, sum == 0.f ? 0.f : v[e] / sum);
}

int attention_ctas(int head_dim, int sm_count) { return sm_count * (head_dim == 256 ? 2 : 3); }

template <int D, int G>
cudaError_t launch(const Kv4AttentionParams& p, int dtype, int sm_count, cudaStream_t st) {
  const size_t smem = (size_t)kWarps * kStages * Stage<D, G>::kBytes;
  if (smem > 48 * 1024) {
    cudaError_t e = cudaFuncSetAttribute(kv4_attention_kernel<D, G>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)smem);
    if (e != cudaSuccess) return e;
  }
  const int ctas = attention_ctas(D, sm_count);
  kv4_attention_kernel<D, G><<<ctas, kThreads, smem, st>>>(p, dtype);
  kv4_join_kernel<D><<<ctas, kRows * 32, 0, st>>>(p, dtype);
  return cudaGetLastError();
}

}  // namespace

size_t kv4_attention_workspace(int head_dim, int sm_count) {
  return (size_t)attention_ctas(head_dim, sm_count) * (sizeof(Part) + 2 * part_bytes(head_dim));
}

cudaError_t launch_kv4_attention(const Kv4AttentionParams& p, int dtype, int sm_count, cudaStream_t st) {
  const int d = p.cache.head_dim, g = p.cache.group;
  if (d == 64) return launch<64, 64>(p, dtype, sm_count, st);
  if (d == 128) return g == 64 ? launch<128, 64>(p, dtype, sm_count, st) : launch<128, 128>(p, dtype, sm_count, st);
  return g == 64 ? launch<256, 64>(p, dtype, sm_count, st) : launch<256, 128>(p, dtype, sm_count, st);
}

}  // namespace tk
