// tk_kv4_attention.cu -- attention over the key/value cache held in 4 bits.
//
// For query i of the n query tokens of a sequence with kv_len tokens in the cache (those n among
// them): o = sum_p w_p v_p, w = softmax_p(scale * q . k_p) over the positions p < kv_len - n + i + 1,
// with k, v = code * scale + offset.  A position whose page is not in the cache counts as absent; a
// query that sees no position gets zeros.
//
// The mathematics.  Scales and offsets stay out of the products (c: codes, per group of dimensions):
//     q . k   = sum_g s_k (q . (c - 8))_g + (m_k + 8 s_k) (sum q)_g
//     sum p v = sum (p s_v) (c - 8)       + sum p (m_v + 8 s_v)
// (Without the shift by 8 the sums carry 7.5 times the sum of the factors, and a long flat softmax
// loses its digits against it.)
// Both products are taken transposed, tokens (dimensions) as the 16 rows of a product, 8 rows of
// queries as its 8 columns, so that no part of the product is idle and a lane holds the sums of two
// rows:  S^T = K Q^T  and  O^T = V^T P^T.
//   Queries against keys: integers.  A row of queries, scaled by a power of two to 22 bits, is three
// signed 8-bit digits, one m16n8k32 product each; the codes are bytes after one AND (and a shift for
// the odd dimensions); the sums are exact.
//   Weights against values: f16.  c - 8 is exact, p s_v is split into two f16 (22 bits), one m16n8k16
// product each.
//   Tiles of four rows (one token of up to four heads a group) put two digits, and both f16 parts of a
// weight, next to each other in the 8 columns: 2 + 1 products instead of 3 + 2, and a lane has half
// the scores (one token of a unit instead of two).
// mma.sync and not tcgen05: one token of a head group is 1 to 8 rows, and tcgen05's operands would have
// to pass through shared memory unpacked (384 bytes a token and head against the 132 that are read).
//
// What bounds it (B200, four heads a group, head dimension 128, group 128): 524288 positions take 128 us,
// 4.5 TB/s of the 6.5 that a copy reaches.  Without its loads the same arithmetic runs at 6.4 TB/s of
// codes, the loads without arithmetic at 5.3, and 12 warps on an SM overlap them only in part; 16 warps
// of 128 registers spill (48 x 4096: 65 us, when 12 took 58; they take 59 now).  A short call is 9 us of waits one after the
// other: lengths, block table, first pages, the end of the tile, the second kernel.
//
// Softmax in base 2 with a running reference per row: w = 2^(s - r) s_v must fit f16, so r follows
// max(s + log2 s_v) and is moved (sums rescaled) only when a weight would leave [0, 2^15].
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <cstdint>
#include <type_traits>

#include "tk_internal.h"
#include "tk_kv4.h"
#include "tk_kv4_attention.cuh"

namespace tk {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kCols = 8;   // columns of a product; a tile has 8 rows (query token, head of the group) or 4
constexpr int kUnit = 16;  // tokens that lie in one page for sure
constexpr int kSub = 2;    // units of a warp's step, which share one reference and its reduction
constexpr int kTokens = kUnit * kSub;
static_assert(kTokens * kWarps == kStep, "");
constexpr int kStages = 2;  // steps of a warp's ring: one computed, one on its way (three: 0 to 4 % slower)
template <int D>
constexpr int kResident = D == 256 ? 2 : 3;  // CTAs of an SM: 255 or 168 registers a thread
constexpr int kFlush = 16;                   // steps between two settings aside of the sums
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16832(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The same, the sum starting at the bits of 1.5 * 2^23: read as f32 it is that plus the sum, while
// the sum is below 2^22 (at most 256 * 15 * 128 here).
constexpr int kSumBits = 0x4B400000;
constexpr float kSumStart = 12582912.f;
__device__ __forceinline__ void mma16832_first(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(kSumBits));
}
// An 8 x 8 matrix of f16, two neighbours of a row a lane, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void ldmatrix_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// Two codes less 8, times 2^-9, from bits 0-3 (codes_lo) or 4-7 (codes_hi) of the halves of x: the
// bits are the subnormals c * 2^-24 and c * 2^-20, and one f16 product and sum of them is exact.
__device__ __forceinline__ uint32_t codes_lo(uint32_t x) {
  uint32_t y;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(y) : "r"(x & 0x000F000Fu), "r"(0x78007800u), "r"(0xA400A400u));  // 2^15, -2^-6
  return y;
}
__device__ __forceinline__ uint32_t codes_hi(uint32_t x) {
  uint32_t y;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(y) : "r"(x & 0x00F000F0u), "r"(0x68006800u), "r"(0xA400A400u));  // 2^11, -2^-6
  return y;
}
constexpr float kCodes = 512.f;  // what undoes the 2^-9

// A stage of a warp's ring: kSub units of 16 tokens' codes and pairs.  Piece c (16 bytes) of a
// token's row lies at c ^ flip(token), so that the 8 rows of an ldmatrix and the lanes of a load of
// keys meet in no bank.
template <int D, int G>
struct Stage {
  static constexpr int NG = D / G;
  static constexpr int kRowBytes = D / 2;
  static constexpr int kPieces = D / 32;
  static constexpr int kCodes = kUnit * kRowBytes;
  static constexpr int kPairs = kUnit * NG * 4;
  static constexpr int kUnitBytes = 2 * (kCodes + kPairs);
  static constexpr int kBytes = kSub * kUnitBytes;
  static __device__ __forceinline__ int flip(int x) {
    return ((x & 1) << 2 | (x & 2) | (x >> 2 & 1)) & (kPieces - 1);
  }
  static __device__ __forceinline__ int at(int token, int byte) {
    return token * kRowBytes + (byte / 16 ^ flip(token)) * 16 + byte % 16;
  }
};

// Shared memory of a CTA: the tile's queries as operands, its rows' numbers, the warps' rings, the
// warps' sums at the end of a tile.
template <int D, int G, int ROWS>
struct Smem {
  using S = Stage<D, G>;
  // [word][lane]: three digits of 32 bits twice, two words idle; of four rows two products' digits twice
  static constexpr int kLaneWords = ROWS == 4 ? 4 : 8;
  static constexpr int kQuery = D / 32 * 32 * kLaneWords * 4;
  static constexpr int kRowWords = 1 + 4 * S::NG;  // unscale; sum, three centres a group
  static constexpr int kRowBytes = kCols * kRowWords * 4;
  static constexpr int kWarp = kStages * S::kBytes;
  static constexpr int kJoint = D + 1;                     // floats of a row of sums at the end
  static constexpr int kJointWarp = kCols * (kJoint + 2);  // and per row the reference and l
  static constexpr int kRings = kQuery + kRowBytes, kJoints = kRings + kWarps * kWarp;
  static constexpr int kBytes = kJoints + kWarps * kJointWarp * 4;
  static_assert(kRowBytes % 16 == 0 && kWarp % 16 == 0, "");
};

template <int D, int G, int ROWS>
__global__ void __launch_bounds__(kThreads, kResident<D>) kv4_attention_kernel(Kv4AttentionParams p, int dtype) {
  using S = Stage<D, G>;
  using M = Smem<D, G, ROWS>;
  constexpr bool kFour = ROWS == 4;
  constexpr int J = kFour ? 1 : 2;  // tokens of a unit that a lane has scores of
  constexpr int NG = S::NG, NT = D / 16;
  extern __shared__ __align__(16) uint8_t smem[];
  // Nothing is read before the kernels before have completed; and nothing through the read-only path
  // (__ldg), which holds only for what no kernel writes once this one has been set up.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int per = p.q_heads / p.cache.kv_heads, hk = p.cache.kv_heads;
  Part* parts = static_cast<Part*>(p.workspace);
  float* sums = reinterpret_cast<float*>(parts + gridDim.x);
  constexpr int kSlot = ROWS * (D + 2);

  // ---- this CTA's run ----
  Run r;
  Tile cur;
  if (!find_run<ROWS, kThreads>(p, per, parts, r, cur)) return;
  const long long run = r.length, start = r.start, stop = r.stop;
  long long at = start;  // of the tile's first step here, in all work

  uint32_t* query = reinterpret_cast<uint32_t*>(smem);
  float* row_num = reinterpret_cast<float*>(smem + M::kQuery);
  uint8_t* ring = smem + M::kRings + warp * M::kWarp;
  const uint32_t ring_addr = (uint32_t)__cvta_generic_to_shared(ring);
  float* joint = reinterpret_cast<float*>(smem + M::kJoints) + warp * M::kJointWarp;
  // the lane's rows, and its token of a unit (and the one 8 on)
  const int my_row = kFour ? 2 * (t & 1) : 2 * t, my_token = kFour ? g + 8 * (t >> 1) : g;
  const bool low = kFour && t >= 2;  // the columns of the lower digit, the lower part of a weight
  // the lane's sum o[i][k] in it: column 2t + k % 2, dimension 32 (i / 2) + 4g + 2 (i % 2) + k / 2
  float* mine_at = joint + 2 * t * M::kJoint + 4 * g;
  auto kept = [&](int i, int k) -> float& {
    return mine_at[(k & 1) * M::kJoint + i / 2 * 32 + i % 2 * 2 + k / 2];
  };

  // where the lane's pieces go in a unit, and where its operands lie
  // (piece 32 i + lane lies 512 i on, at D = 256 with one bit of its place turned for odd i)
  const uint32_t piece_dst = S::at(lane / S::kPieces, lane % S::kPieces * 16);
  const uint32_t pair_dst = 2 * S::kCodes + (lane < 16 ? 0 : S::kPairs) + (lane & 15) * 16;
  int k_at[NG];
#pragma unroll
  for (int y = 0; y < NG; ++y) k_at[y] = S::at(g, y * (G / 2) + t * (G / 8));
  // ldmatrix: lanes 0-7, 8-15 the rows of tokens 0-7, 8-15 at one piece, lanes 16-31 at the next
  const uint32_t v_row = S::kCodes + (lane & 15) * S::kRowBytes, v_piece = (lane >> 4) ^ S::flip(lane & 15);
  const uint32_t page_bytes = (uint32_t)(hk << p.cache.shift) * S::kRowBytes;  // at most 2^16 heads of 2^8 rows of 2^7
  const int page_mask = (1 << p.cache.shift) - 1;
  const ptrdiff_t k_to_v = p.cache.v_codes - p.cache.k_codes;

  // ---- queue of loads of a tile: a unit is four runs of consecutive bytes ----
  const uint8_t *k_src, *pair_src;  // of the head in page 0, and the lane's piece
  const int* table;
  int s0, s1, see_most, page[kSub];
  unsigned valid = 0;  // kSub bits a stage
  auto look = [&](int step) {
#pragma unroll
    for (int u = 0; u < kSub; ++u) {
      const int pos = step * kStep + warp * kTokens + u * kUnit;
      page[u] = step < s1 && pos < see_most ? table[pos >> p.cache.shift] : -1;
    }
  };
  auto issue = [&](int stage, int step) {
#pragma unroll
    for (int u = 0; u < kSub; ++u) {
      const unsigned bit = 1u << (stage * kSub + u);
      valid &= ~bit;
      if ((unsigned)page[u] < (unsigned)p.cache.num_blocks) {
        valid |= bit;
        const int pos = step * kStep + warp * kTokens + u * kUnit;
        const uint64_t codes = (uint64_t)(uint32_t)page[u] * page_bytes + (uint32_t)((pos & page_mask) * S::kRowBytes);
        const uint32_t dst = ring_addr + stage * S::kBytes + u * S::kUnitBytes;
        const uint32_t dst0 = dst + piece_dst, dst1 = dst + (D == 256 ? piece_dst ^ 16 : piece_dst);
        const uint8_t *kc = k_src + codes, *vc = kc + k_to_v;
#pragma unroll
        for (int i = 0; i < S::kCodes / 512; ++i) {
          cp_async16((i & 1 ? dst1 : dst0) + i * 512, kc + i * 512);
          cp_async16((i & 1 ? dst1 : dst0) + S::kCodes + i * 512, vc + i * 512);
        }
        if ((lane & 15) < 4 * NG) cp_async16(dst + pair_dst, pair_src + codes / (S::kRowBytes / NG / 4));
      }
    }
    cp_commit();
  };
  // a row's query token of its sequence; a row is (token, head of the group)
  auto token_of = [&](const Tile& x, int row) { return x.s.n == 1 ? 0 : row / per; };
  // the position after the last that row r of a tile sees; its last row sees most, its first least
  auto sees = [&](const Tile& x, int r) {
    const int row = x.rt * ROWS + r, end = x.s.n * per - 1;
    return min(x.s.kv, x.s.last + token_of(x, min(row, end)) + 1);
  };
  constexpr int LPR = D / 8;                                   // threads of a row of queries, 8 dimensions each
  constexpr int kPasses = (ROWS * LPR + kThreads - 1) / kThreads;
  float q[kPasses][8];
  auto begin = [&](const Tile& x) {
    const uint64_t head_at = (uint64_t)(uint32_t)(x.head << p.cache.shift) * S::kRowBytes;
    k_src = p.cache.k_codes + head_at + lane * 16;
    pair_src = reinterpret_cast<const uint8_t*>(lane < 16 ? p.cache.k_scales : p.cache.v_scales) +
               head_at / (S::kRowBytes / NG / 4) + (lane & 15) * 16;
    table = p.block_tables + (size_t)x.b * p.max_blocks;
    s0 = max(x.c0 - kTileCost, 0);
    s1 = max(x.c1 - kTileCost, 0);
    see_most = sees(x, ROWS - 1);
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int r = i * (kThreads / LPR) + tid / LPR;
      const int row = min(x.rt * ROWS + r, x.s.n * per - 1);
#pragma unroll
      for (int k = 0; k < 8; ++k) q[i][k] = 0.f;
      const int token = token_of(x, row);
      if (r < ROWS && sees(x, r) > 0)
        load_row8(p.q, (long long)(x.s.first + token) * p.q_stride + (long long)(x.head * per + row - token * per) * D +
                           tid % LPR * 8, dtype, q[i]);
    }
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) {
      look(s0 + i);
      issue(i, s0 + i);
    }
    look(s0 + kStages - 1);
  };
  begin(cur);

  for (;;) {
      const int see_least = sees(cur, 0), see[2] = {sees(cur, my_row), sees(cur, my_row + 1)};

      // ---- queries: scaled, as integers of 22 bits, in digits; 8 dimensions a thread ----
#pragma unroll
      for (int pass = 0; pass < kPasses; ++pass) {
        const int r = pass * (kThreads / LPR) + tid / LPR, at8 = tid % LPR;
        if (r >= ROWS) continue;  // whole warps
        const float f = p.scale * 1.4426950408889634f;
        float top = 0.f, odd = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          q[pass][i] *= f;
          top = fmaxf(top, fabsf(q[pass][i]));
          odd = fmaf(q[pass][i], 0.f, odd);  // NaN if one is not finite
        }
#pragma unroll
        for (int off = LPR / 2; off > 0; off >>= 1) {
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
          odd += __shfl_xor_sync(0xffffffffu, odd, off);
        }
        // the largest becomes 2^21 .. 2^22
        const int e = top > 0.f && top < INFINITY ? min(21 - ilogbf(top), 120) : 0;
        const float norm = ldexpf(1.f, e);
        float sum = 0.f;
        int sums[3] = {};  // of the digits
        uint32_t digits[3][2] = {};  // highest first; of the even, the odd dimensions
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          int x = __float2int_rn(q[pass][i] * norm);
          sum += (float)x;
          const int d0 = (int8_t)x;
          x = (x - d0) >> 8;
          const int d1 = (int8_t)x;
          x = (x - d1) >> 8;
          sums[0] += x;
          sums[1] += d1;
          sums[2] += d0;
          digits[0][i & 1] |= (uint32_t)(x & 255) << (i / 2 * 8);
          digits[1][i & 1] |= (uint32_t)(d1 & 255) << (i / 2 * 8);
          digits[2][i & 1] |= (uint32_t)(d0 & 255) << (i / 2 * 8);
        }
#pragma unroll
        for (int off = G / 16; off > 0; off >>= 1) {
          sum += __shfl_xor_sync(0xffffffffu, sum, off);
#pragma unroll
          for (int d = 0; d < 3; ++d) sums[d] += __shfl_xor_sync(0xffffffffu, sums[d], off);
        }
        const int y = at8 / (G / 8), tt = at8 % (G / 8) / (G / 32), w = y * (G / 32) + at8 % (G / 32);
        uint32_t* dst = query + (w * 32 + r * 4 + tt) * M::kLaneWords;
        if constexpr (kFour) {  // columns 0-3, 4-7: the highest digit, the next; the lowest twice
          *reinterpret_cast<uint4*>(dst) = make_uint4(digits[0][0], digits[0][1], digits[2][0], digits[2][1]);
          *reinterpret_cast<uint4*>(dst + 16 * M::kLaneWords) =
              make_uint4(digits[1][0], digits[1][1], digits[2][0], digits[2][1]);
        } else {
          *reinterpret_cast<uint4*>(dst) = make_uint4(digits[0][0], digits[0][1], digits[1][0], digits[1][1]);
          *reinterpret_cast<uint2*>(dst + 4) = make_uint2(digits[2][0], digits[2][1]);
        }
        float* num = row_num + r * M::kRowWords;
        if (at8 == 0) num[0] = ldexpf(1.f, -e) + odd;
        if (at8 % (G / 8) == 0) {
          num[1 + 4 * y] = sum;
#pragma unroll
          for (int d = 0; d < 3; ++d) num[2 + 4 * y + d] = kSumStart + (float)(8 * sums[d]);
        }
      }
      __syncthreads();
      // of the lane's two rows
      float unscale[2], qsum[NG][2], off_sum[NG][2], l[2] = {0.f, 0.f};
      float ref[2] = {-INFINITY, -INFINITY};  // weights are 2^(s - ref + 10) s_v
      float centre[NG][3][2];                 // where a digit's sum begins, and 8 times the sum of the row's digits
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float* num = row_num + (my_row + i) * M::kRowWords;
        unscale[i] = num[0];
#pragma unroll
        for (int y = 0; y < NG; ++y) {
          qsum[y][i] = num[1 + 4 * y];
#pragma unroll
          for (int d = 0; d < 3; ++d) centre[y][d][i] = num[2 + 4 * y + d];
          // four rows: of the lane's own digit, at its place; exact, so that a product and sum with it is
          if (kFour) centre[y][0][i] = low ? -256.f * num[3 + 4 * y] : -65536.f * num[2 + 4 * y];
          off_sum[y][i] = 0.f;
        }
      }
      const float place = low ? 256.f : 65536.f;  // of the lane's digit
      // sums: products of 16 dimensions, 32 z + 4 g + 2 h + {0, 1} in o[2 z + h], of columns 2t, 2t + 1
      float o[NT][4];
#pragma unroll
      for (int i = 0; i < NT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
      // Sums set aside, in the warp's place for the join: O with off_sum in it, and l behind it
      bool flushed = false;
      int since = 0;  // steps since then
      auto aside_l = [&](int row) -> float& { return joint[(my_row + row) * M::kJoint + D]; };
      auto sum_lanes = [&] {  // of a row, what they have of l and off_sum
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int off = kFour ? 2 : 4; off < 32; off <<= 1) {
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], off);
#pragma unroll
            for (int y = 0; y < NG; ++y) off_sum[y][i] += __shfl_xor_sync(0xffffffffu, off_sum[y][i], off);
          }
      };

      // ---- the steps ----
      int stage = 0;
      for (int step = s0; step < s1; ++step) {
        cp_wait<kStages - 2>();
        __syncwarp();
        const unsigned there = valid >> (stage * kSub) & ((1u << kSub) - 1);
        issue(stage == 0 ? kStages - 1 : stage - 1, step + kStages - 1);
        look(step + kStages);
        const uint8_t* st = ring + stage * S::kBytes;
        stage = stage == kStages - 1 ? 0 : stage + 1;
        if (!there) continue;
        const int pos = step * kStep + warp * kTokens;

        // Two forms of a step: one masks what a row does not see
        auto step_of = [&](auto masked) {
        constexpr bool kMasked = decltype(masked)::value;

        // scores of the lane's tokens of the units against its rows, in units of unscale
        float sc[kSub][J][2], vs[kSub][J][NG], vm[kSub][J][NG], top[2] = {-INFINITY, -INFINITY};
        unsigned hidden = 0;  // scores that are not seen
#pragma unroll
        for (int u = 0; u < kSub; ++u) {
          const uint8_t* su = st + u * S::kUnitBytes;
          const uint32_t* pairs = reinterpret_cast<const uint32_t*>(su + 2 * S::kCodes) + my_token * NG;
          float lg[J];
#pragma unroll
          for (int j = 0; j < J; ++j) {
            float most = 5.9604645e-8f;  // 2^-24, the least f16
#pragma unroll
            for (int y = 0; y < NG; ++y) {
              const uint32_t pair = pairs[(kUnit + j * 8) * NG + y];
              vs[u][j][y] = half_lo(pair);
              vm[u][j][y] = fmaf(vs[u][j][y], 8.f, half_hi(pair));
              most = fmaxf(most, fabsf(vs[u][j][y]));
            }
            lg[j] = lg2(most);
            sc[u][j][0] = sc[u][j][1] = 0.f;
          }
#pragma unroll
          for (int y = 0; y < NG; ++y) {
            uint32_t w[2][G / 32];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const uint8_t* src = su + k_at[y] + j * 8 * S::kRowBytes;
              if constexpr (G == 128)
                *reinterpret_cast<uint4*>(w[j]) = *reinterpret_cast<const uint4*>(src);
              else
                *reinterpret_cast<uint2*>(w[j]) = *reinterpret_cast<const uint2*>(src);
            }
            constexpr int P = kFour ? 2 : 3;  // products
            int c[P][4];
#pragma unroll
            for (int i = 0; i < G / 32; ++i) {
              // the digits of column g: from shared memory again, for the registers' sake
              const uint32_t* qs = query + ((y * (G / 32) + i) * 32 + lane) * M::kLaneWords;
              const uint4 q4 = *reinterpret_cast<const uint4*>(qs);
              uint32_t qd[P][2];
              qd[0][0] = q4.x, qd[0][1] = q4.y, qd[1][0] = q4.z, qd[1][1] = q4.w;
              if constexpr (!kFour) {
                const uint2 q2 = *reinterpret_cast<const uint2*>(qs + 4);
                qd[2][0] = q2.x, qd[2][1] = q2.y;
              }
              const uint32_t a[4] = {w[0][i] & 0x0F0F0F0Fu, w[1][i] & 0x0F0F0F0Fu, w[0][i] >> 4 & 0x0F0F0F0Fu,
                                     w[1][i] >> 4 & 0x0F0F0F0Fu};
#pragma unroll
              for (int d = 0; d < P; ++d) {
                if (i == 0)
                  mma16832_first(c[d], a, qd[d][0], qd[d][1]);
                else
                  mma16832(c[d], a, qd[d][0], qd[d][1]);
              }
            }
            if constexpr (kFour) {
              const uint32_t pair = pairs[y];
              const float ks = half_lo(pair), km = fmaf(ks, 8.f, half_hi(pair));
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                // the lane's digit of both tokens, at its place: exact.  The lane two on (mod 4) has the other
                const float x0 = fmaf(__int_as_float(c[0][i]), place, centre[y][0][i]);
                const float x8 = fmaf(__int_as_float(c[0][2 + i]), place, centre[y][0][i]);
                float dot = __int_as_float(low ? c[1][2 + i] : c[1][i]) - centre[y][2][i];
                dot += (low ? x8 : x0) + __shfl_xor_sync(0xffffffffu, low ? x0 : x8, 2);
                sc[u][0][i] = fmaf(dot, ks, fmaf(qsum[y][i], km, sc[u][0][i]));
              }
            } else {
#pragma unroll
              for (int j = 0; j < J; ++j) {
                const uint32_t pair = pairs[j * 8 * NG + y];
                const float ks = half_lo(pair), km = fmaf(ks, 8.f, half_hi(pair));
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                  float dot = __int_as_float(c[0][2 * j + i]) - centre[y][0][i];  // exact, as the next two
                  dot = fmaf(dot, 256.f, __int_as_float(c[1][2 * j + i]) - centre[y][1][i]);
                  dot = fmaf(dot, 256.f, __int_as_float(c[P - 1][2 * j + i]) - centre[y][2][i]);
                  sc[u][j][i] = fmaf(dot, ks, fmaf(qsum[y][i], km, sc[u][j][i]));
                }
              }
            }
          }
          if constexpr (kMasked) {  // of what a row does not see nothing counts, and it may be NaN
#pragma unroll
            for (int j = 0; j < J; ++j) {
              const int at_token = there >> u & 1 ? pos + u * kUnit + j * 8 + my_token : 0x7fffffff;
              if (at_token >= see_most) {
#pragma unroll
                for (int y = 0; y < NG; ++y) vs[u][j][y] = vm[u][j][y] = 0.f;
              }
#pragma unroll
              for (int i = 0; i < 2; ++i)
                if (at_token >= see[i]) {
                  sc[u][j][i] = -INFINITY;
                  hidden |= 1u << (4 * u + 2 * j + i);
                }
            }
          }
          // reference: the row's largest s + log2 of the value scale
#pragma unroll
          for (int j = 0; j < J; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) top[i] = fmaxf(top[i], fmaf(sc[u][j][i], unscale[i], lg[j]));
        }
        if (__any_sync(0xffffffffu, top[0] > ref[0] + 5.f || top[1] > ref[1] + 5.f)) {
#pragma unroll
          for (int off = kFour ? 2 : 4; off < 32; off <<= 1) {
            top[0] = fmaxf(top[0], __shfl_xor_sync(0xffffffffu, top[0], off));
            top[1] = fmaxf(top[1], __shfl_xor_sync(0xffffffffu, top[1], off));
          }
          const bool move0 = top[0] > ref[0] + 5.f, move1 = top[1] > ref[1] + 5.f;
          const float f0 = move0 ? ex2(ref[0] - top[0]) : 1.f, f1 = move1 ? ex2(ref[1] - top[1]) : 1.f;  // 0 at first
          if (move0) ref[0] = top[0];
          if (move1) ref[1] = top[1];
          l[0] *= f0;
          l[1] *= f1;
#pragma unroll
          for (int y = 0; y < NG; ++y) {
            off_sum[y][0] *= f0;
            off_sum[y][1] *= f1;
          }
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            o[i][0] *= f0;
            o[i][1] *= f1;
            o[i][2] *= f0;
            o[i][3] *= f1;
          }
          if (flushed) {
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
              for (int k = 0; k < 4; ++k) kept(i, k) *= k & 1 ? f1 : f0;
            if (g == 0 && !low) {
              aside_l(0) *= f0;
              aside_l(1) *= f1;
            }
          }
        }
        const float base[2] = {ref[0] == -INFINITY ? 0.f : 10.f - ref[0], ref[1] == -INFINITY ? 0.f : 10.f - ref[1]};

#pragma unroll
        for (int u = 0; u < kSub; ++u) {
          float pr[J][2];
#pragma unroll
          for (int j = 0; j < J; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              pr[j][i] = ex2(fmaf(sc[u][j][i], unscale[i], base[i]));
              l[i] += pr[j][i];
            }
#pragma unroll
          for (int y = 0; y < NG; ++y) {
            uint32_t hi[2], lo[2];  // four rows: hi holds both parts
#pragma unroll
            for (int j = 0; j < J; ++j) {
              float w[2];
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                w[i] = pr[j][i] * vs[u][j][y];
                const float with = fmaf(pr[j][i], vm[u][j][y], off_sum[y][i]);
                if (!(kMasked && hidden >> (4 * u + 2 * j + i) & 1))
                  off_sum[y][i] = with;
                else
                  w[i] = 0.f;
              }
              split_f16(w[0], w[1], hi[j], lo[j]);
            }
            if constexpr (kFour) {
              // columns 0-3 the upper parts of tokens 0-7 (8-15), columns 4-7 the lower ones
              const uint32_t other = __shfl_xor_sync(0xffffffffu, low ? hi[0] : lo[0], 2);
              const uint32_t m0 = low ? other : hi[0], m8 = low ? lo[0] : other;
              hi[0] = transpose8(m0);
              hi[1] = transpose8(m8);
            } else {
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                hi[j] = transpose8(hi[j]);  // tokens 8j + 2t, 8j + 2t + 1 of row g
                lo[j] = transpose8(lo[j]);
              }
            }
#pragma unroll
            for (int z = y * (G / 32); z < (y + 1) * (G / 32); z += 2) {  // 32 dimensions each
              uint32_t c[4];  // of 4 dimensions: tokens 2t, 2t + 1; 8 + 2t, 9 + 2t; then of the next 32
              ldmatrix_trans(c, ring_addr + (uint32_t)(st - ring) + u * S::kUnitBytes + v_row + (v_piece ^ z) * 16);
              uint32_t a[4][4];
#pragma unroll
              for (int h = 0; h < 4; ++h) {
                uint32_t x = c[h / 2 * 2], x8 = c[h / 2 * 2 + 1];
                if (h & 1) x >>= 8, x8 >>= 8;
                a[h][0] = codes_lo(x), a[h][1] = codes_hi(x), a[h][2] = codes_lo(x8), a[h][3] = codes_hi(x8);
                mma16816(o[2 * z + h], a[h], hi[0], hi[1]);
              }
              if constexpr (!kFour) {
#pragma unroll
                for (int h = 0; h < 4; ++h) mma16816(o[2 * z + h], a[h], lo[0], lo[1]);
              }
            }
          }
        }
        };
        if (there != (1u << kSub) - 1 || pos + kTokens > see_least)
          step_of(std::true_type{});
        else
          step_of(std::false_type{});
        // The tensor core drops what lies under the last bit of a sum, always towards 0, and f32 additions of
        // equal weights round the same way each time: the sums are set aside before that adds up, each time
        // starting with what the addition dropped (f32 outputs of one CTA, 8192 positions: 2.8e-6 off without it;
        // 131072 equal tokens: 24e-6 with l and off_sum as running sums, now 1e-6, as over 2048; costs 2 %).
        if (++since == kFlush) {
          since = 0;
          sum_lanes();
#pragma unroll
          for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float x = low ? o[i][k] * kCodes : fmaf(o[i][k], kCodes, off_sum[i / (G / 16)][k & 1]);
              o[i][k] = keep(flushed, kept(i, k), 1.f, x) * (1.f / kCodes);
            }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            l[i] = g == 0 && !low ? keep(flushed, aside_l(i), 1.f, l[i]) : 0.f;
#pragma unroll
            for (int y = 0; y < NG; ++y) off_sum[y][i] = 0.f;
          }
          flushed = true;
        }
      }
      cp_wait<0>();
      __syncwarp();

      // ---- join the four warps ----
      sum_lanes();
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float x = low ? o[i][k] * kCodes : fmaf(o[i][k], kCodes, off_sum[i / (G / 16)][k & 1]);
          if (flushed) x += kept(i, k);
          if (kFour) x += __shfl_xor_sync(0xffffffffu, x, 2);  // both parts
          if (!low) kept(i, k) = x;
        }
      if (g == 0 && !low) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          joint[kCols * M::kJoint + 2 * (my_row + i)] = ref[i];
          joint[kCols * M::kJoint + 2 * (my_row + i) + 1] = flushed ? l[i] + aside_l(i) : l[i];
        }
      }

      // the next tile's first loads travel meanwhile
      const Tile done = cur;
      const long long done_at = at;
      at += cur.c1 - cur.c0;
      const bool more = at < stop;
      if (more) {
        next_tile<ROWS>(p, per, at, stop, cur);
        begin(cur);
      }
      __syncthreads();

      {
        const bool whole = done.c0 == 0 && done.c1 == done.steps;
        const int row0 = done.rt * ROWS, rows = min(ROWS, done.s.n * per - row0), slot = done_at == start ? 0 : 1;
        constexpr int kThreadsRow = kThreads / ROWS;
        const int row = tid / kThreadsRow, d0 = tid % kThreadsRow;
        const float* all = reinterpret_cast<const float*>(smem + M::kJoints);
        const float* num = all + kCols * M::kJoint + 2 * row;
        float top = -INFINITY, sum = 0.f, f[kWarps];
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, num[w * M::kJointWarp]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float r = num[w * M::kJointWarp];
          f[w] = r == -INFINITY ? 1.f : ex2(r - top);  // no reference: sums of 0, or of NaN
          sum = fmaf(num[w * M::kJointWarp + 1], f[w], sum);
        }
        float* out = sums + ((size_t)blockIdx.x * 2 + slot) * kSlot;
        const int query_row = row0 + min(row, rows - 1);
        const int token = token_of(done, query_row);
        const long long o_at = (long long)(done.s.first + token) * p.o_stride +
                               (long long)(done.head * per + query_row - token * per) * D;
#pragma unroll
        for (int d = d0; d < D; d += kThreadsRow) {
          float v = 0.f;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) v = fmaf(all[w * M::kJointWarp + row * M::kJoint + d], f[w], v);
          if (!whole)
            out[row * D + d] = v;
          else if (row < rows)
            store_any(p.o, o_at + d, dtype, sum == 0.f ? 0.f : v / sum);
        }
        if (!whole && d0 == 0) {
          out[ROWS * D + 2 * row] = top;
          out[ROWS * D + 2 * row + 1] = sum;
        }
        if (!whole && done.c0 == 0 && tid == 0) {  // the tile begins here: where its parts are
          const long long end = done_at + done.steps;
          parts[blockIdx.x] =
              Part{done.s.first, rows, done.head, (int)((end - 1) / run - blockIdx.x + 1), row0, slot, 0, 0};
        }
      }
      if (!more) break;
  }
}

// Rows of a tile: four where a sequence has as many on the mean (its own query tokens are not known
// here), eight otherwise: with four heads a group, 48 x 4096 59 us instead of 68, 524288 128 instead of
// 146; with eight, four-row tiles would read the cache twice.
int attention_rows(const Kv4AttentionParams& p) {
  const long long per = p.q_heads / p.cache.kv_heads;
  return p.tokens * per <= 4ll * p.batch ? 4 : 8;
}

int attention_ctas(int head_dim, int sm_count) { return sm_count * (head_dim == 256 ? kResident<256> : kResident<128>); }

template <int D, int G, int ROWS>
cudaError_t launch(Kv4AttentionParams p, int dtype, int sm_count, cudaStream_t st) {
  const size_t smem = Smem<D, G, ROWS>::kBytes;
  // shared memory above 48 KB is asked for once per device (and again in a new context of it)
  constexpr int kMaxDevices = 64;
  static std::atomic<unsigned> asked[kMaxDevices];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const unsigned gen = attr_generation(dev) + 1;
  if (dev >= kMaxDevices || asked[dev].load(std::memory_order_acquire) != gen) {
    e = cudaFuncSetAttribute(kv4_attention_kernel<D, G, ROWS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    if (dev < kMaxDevices) asked[dev].store(gen, std::memory_order_release);
  }
  // programmatic launches: a kernel is set up while the one before it runs, and passes its wait when
  // that has completed
  const int ctas = attention_ctas(D, sm_count);
  p.inv_ctas = 1.0 / ctas;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kv4_attention_kernel<D, G, ROWS>, p, dtype);
  if (e != cudaSuccess) return e;
  cfg.dynamicSmemBytes = 0;
  // Parts that a tile may have, by the table's reach and the CTAs: many want more warps a row (1 x 131072,
  // 56 parts: 3.8 us with 4, 2.3 with 8; 8 x 2000, 7 parts: 0.6 us less with 4), many tiles want fewer
  // CTAs, most of which have nothing to do (48 x 4096: 1 us less with four rows a CTA than with two).
  const long long tiles = ((long long)p.tokens * (p.q_heads / p.cache.kv_heads) / ROWS + p.batch) * p.cache.kv_heads;
  const long long steps = (((long long)p.max_blocks << p.cache.shift) + kStep - 1) / kStep + kTileCost;
  if (tiles <= sm_count && std::min(steps, ctas / tiles) > 16) {
    cfg.gridDim = dim3((unsigned)ctas, ROWS / 2);
    cfg.blockDim = dim3(2 * 8 * 32);
    return cudaLaunchKernelEx(&cfg, kv4_join_kernel<D, ROWS, 2, 8>, p, dtype);
  }
  if (tiles <= sm_count) {
    cfg.gridDim = dim3((unsigned)ctas, ROWS / 2);
    cfg.blockDim = dim3(2 * 4 * 32);
    return cudaLaunchKernelEx(&cfg, kv4_join_kernel<D, ROWS, 2, 4>, p, dtype);
  }
  cfg.gridDim = dim3((unsigned)ctas, ROWS / 4);
  cfg.blockDim = dim3(4 * 2 * 32);
  return cudaLaunchKernelEx(&cfg, kv4_join_kernel<D, ROWS, 4, 2>, p, dtype);
}

}  // namespace

size_t kv4_attention_workspace(int head_dim, int sm_count) {
  return std::max(attention_workspace(attention_ctas(head_dim, sm_count), kCols, head_dim),
                  kv4_prompt_workspace(head_dim, sm_count));
}

cudaError_t launch_kv4_attention(const Kv4AttentionParams& p, int dtype, int sm_count, cudaStream_t st) {
  const int d = p.cache.head_dim, g = p.cache.group;
  if (kv4_prompt_takes(p, dtype)) return launch_kv4_prompt(p, dtype, sm_count, st);
  if (attention_rows(p) == 4) {
    if (d == 64) return launch<64, 64, 4>(p, dtype, sm_count, st);
    if (d == 128) return g == 64 ? launch<128, 64, 4>(p, dtype, sm_count, st) : launch<128, 128, 4>(p, dtype, sm_count, st);
    return g == 64 ? launch<256, 64, 4>(p, dtype, sm_count, st) : launch<256, 128, 4>(p, dtype, sm_count, st);
  }
  if (d == 64) return launch<64, 64, 8>(p, dtype, sm_count, st);
  if (d == 128) return g == 64 ? launch<128, 64, 8>(p, dtype, sm_count, st) : launch<128, 128, 8>(p, dtype, sm_count, st);
  return g == 64 ? launch<256, 64, 8>(p, dtype, sm_count, st) : launch<256, 128, 8>(p, dtype, sm_count, st);
}

}  // namespace tk
