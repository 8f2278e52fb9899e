// tk_kv4_prompt.cu -- attention over the 4-bit cache for many query rows a key head: prompts and
// their chunks.
//
// The mathematics is that of tk_kv4_attention.cu, with one group a head and queries of 16 bits, and
// the products on tcgen05: a tile is 128 rows (query token, head of the group) against 128 tokens a
// step.
//   S = Q (c - 8)^T    Q as it is (f16 or bf16), the codes exact in either
//   t = a S + b sum(q) + log2 |s_v|      a = f s_k, b = f (m_k + 8 s_k), f = scale log2 e
//   w = 2^(t - r),  O += w sign(s_v) (c - 8),  l += w / |s_v|,  off += w (m_v + 8 s_v) / |s_v|
// and o = (O + off) / l.  So a weight comes out of the exponential with its scale in it, ready for
// the second product; it is split into two f16 (22 bits), two products into one accumulator.
// s_v = 0 counts as 1 with values of 0.  A row's reference r keeps the weights below 2^15; when one
// would pass, r is moved so that the largest is 2^10, and the sums are rescaled, which is rare.
//
// One CTA is 256 threads, two a row: tokens 0-63 and 64-127 of a step, and half of the dimensions of
// O.  Tensor memory: S (128 columns), over which the weights lie as f16 pairs once all of S has been
// read, and O.  A step is one chain (unpack keys, S, weights, O), so two CTAs live on an SM, one
// computing while the other's products run.  Warps wait for products, the two of a row for each other,
// and one, which issues the products, for all.  The next step's codes travel meanwhile: those of keys
// into the operand's own rows, whose products have completed.
//   The tensor core's sums round toward zero: O is set aside into the CTA's slot of the workspace, in
// f32 additions, every kFlush steps.
//
// What bounds it (B200; 2 x 256 tokens over 1500 to 4000 positions, 40 + 8 heads of 128, bf16): 112 us,
// 290 TFLOP/s with one product each (the second part of the weights is a third one); tiles of eight rows
// on mma.sync take 299.  Instruction issue and its latencies: 1400 instructions a warp and step at 0.47 a
// cycle and scheduler, four warps a scheduler (128 registers, most of them scores), tensor pipe 24 %
// busy.  Numbers of tokens for eight instead of four columns at a time: 125 us, spilled.  One f16 part of
// a weight instead of two: 102 us, but 11 bits.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "tk_internal.h"
#include "tk_kv4_attention.cuh"
#include "tk_ptx.cuh"

namespace tk {
namespace {

constexpr int kRows = 128, kThreads = 256, kFlush = 16, kCtasPerSm = 2;
constexpr uint32_t kTmemCols = 256, kTmemO = 128, kTmemLow = 64;  // S and the weights' high parts at 0
constexpr unsigned kErrWait = 4u;                                  // a product never completed

// Waits, a warp together, for the phase of `bar`; gives up, for good, after timeout_ns.
__device__ __forceinline__ void wait_phase(uint64_t* bar, uint32_t phase, bool& dead, const Kv4AttentionParams& p) {
  if (!dead && !mbar_try_wait(bar, phase)) {
    const uint64_t t0 = global_timer_ns();
    while (!mbar_try_wait(bar, phase))
      if (global_timer_ns() - t0 > p.timeout_ns) {
        atomicOr(p.err, kErrWait);
        dead = true;
        break;
      }
  }
  __syncwarp();
  tcgen05_fence_after();
}

#define TK_R4(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3])
#define TK_R16(r, i) TK_R4(r, i), TK_R4(r, i + 4), TK_R4(r, i + 8), TK_R4(r, i + 12)
#define TK_V4(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3])
// 64 (16) consecutive columns of the warp's 32 lanes, complete on return.
__device__ __forceinline__ void tmem_load64(uint32_t at, uint32_t (&r)[64]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, %34, %35, "
      "%36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, "
      "%57, %58, %59, %60, %61, %62, %63}, [%64];\n\ttcgen05.wait::ld.sync.aligned;"
      : TK_R16(r, 0), TK_R16(r, 16), TK_R16(r, 32), TK_R16(r, 48)
      : "r"(at)
      : "memory");
}
__device__ __forceinline__ void tmem_load16(uint32_t at, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15}, [%16];\n\ttcgen05.wait::ld.sync.aligned;"
      : TK_R16(r, 0)
      : "r"(at)
      : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t at, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16};" ::"r"(at),
      TK_V4(r, 0), TK_V4(r, 4), TK_V4(r, 8), TK_V4(r, 12)
      : "memory");
}
#undef TK_R4
#undef TK_R16
#undef TK_V4

// Eight codes less 8 from a word of them, times m: f16, or bf16 (m = 1).  The bits 0x6400 | c are the
// f16 1024 + c, 0x4300 | c the bf16 128 + c; both differences are exact.
__device__ __forceinline__ uint4 codes_f16(uint32_t w, uint32_t m, uint32_t shift) {  // shift: -1032 m
  const uint32_t w4 = w >> 4;
  uint32_t y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t x = (__byte_perm(w, w4, 0x4400 + i * 0x1111) & 0x000F000Fu) | 0x64006400u;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(y[i]) : "r"(x), "r"(m), "r"(shift));
  }
  return make_uint4(y[0], y[1], y[2], y[3]);
}
__device__ __forceinline__ uint4 codes_bf16(uint32_t w) {
  const uint32_t w4 = w >> 4;
  uint32_t y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t x = (__byte_perm(w, w4, 0x4400 + i * 0x1111) & 0x000F000Fu) | 0x43004300u;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(y[i]) : "r"(x), "r"(0x3F803F80u), "r"(0xC308C308u));  // 1, -136
  }
  return make_uint4(y[0], y[1], y[2], y[3]);
}

__device__ __forceinline__ uint4 load_bits8(const uint16_t* src) {
  if (reinterpret_cast<uintptr_t>(src) % 16 == 0) return *reinterpret_cast<const uint4*>(src);
  uint32_t w[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) w[k] = src[2 * k] | (uint32_t)src[2 * k + 1] << 16;
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void store_bits8(uint16_t* dst, const uint4& y) {
  if (reinterpret_cast<uintptr_t>(dst) % 16 == 0) {
    *reinterpret_cast<uint4*>(dst) = y;
    return;
  }
  const uint32_t w[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
  for (int k = 0; k < 8; ++k) dst[k] = (uint16_t)(w[k / 2] >> (k % 2 * 16));
}
__device__ __forceinline__ void add_scaled(float4& x, const float4& y, float f) {
  x.x = fmaf(y.x, f, x.x);
  x.y = fmaf(y.y, f, x.y);
  x.z = fmaf(y.z, f, x.z);
  x.w = fmaf(y.w, f, x.w);
}
template <bool BF>
__device__ __forceinline__ uint32_t pack_out(float a, float b) {
  if constexpr (!BF) return pack_f16(a, b);
  uint32_t y;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(b), "f"(a));
  return y;
}

__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Two f32 at once.
struct Pair {
  unsigned long long x;
};
__device__ __forceinline__ Pair pair_of(float a, float b) {
  Pair y;
  asm("mov.b64 %0, {%1, %2};" : "=l"(y.x) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float2 values_of(Pair p) {
  float2 y;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(y.x), "=f"(y.y) : "l"(p.x));
  return y;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair y;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(y.x) : "l"(a.x), "l"(b.x), "l"(c.x));
  return y;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair y;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(y.x) : "l"(a.x), "l"(b.x));
  return y;
}
__device__ __forceinline__ void load_pairs(const float* src, Pair (&y)[2]) {  // 4 floats on a 16-byte boundary
  const float4 v = *reinterpret_cast<const float4*>(src);
  y[0] = pair_of(v.x, v.y);
  y[1] = pair_of(v.z, v.w);
}

// Operands in shared memory: rows of 64 values (128 bytes), their 16-byte pieces turned by the row's
// number; heads of 128 dimensions as two halves.  Keys and queries [half][row], values by eights of
// tokens [token / 8][half][token % 8].
template <int D>
struct PromptSmem {
  static constexpr int kOperand = kRows * D * 2;
  static constexpr int kQ = 0, kK = kOperand, kV = 2 * kOperand, kRaw = 3 * kOperand, kNums = kRaw + kStep * D / 2;
  // per token, twice, a, b, log2 |s_v|, 1 / |s_v|, (m_v + 8 s_v) / |s_v|; per row sum(q), and two halves' numbers twice
  static constexpr int kBytes = kNums + (2 * 5 * kStep + kRows + 4 * kRows) * 4 + 1024;
};

template <int D, bool BF>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) kv4_prompt_kernel(Kv4AttentionParams p) {
  using M = PromptSmem<D>;
  constexpr int H = D / 64;          // halves of a head, 128 bytes a row
  constexpr int kWords = D / 16;     // of codes of half a head
  extern __shared__ uint8_t dynamic[];
  __shared__ uint64_t bar, keys_bar, weights_bar;  // products complete; all warps' keys, weights written
  __shared__ uint32_t tmem_slot;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int per = p.q_heads / p.cache.kv_heads, hk = p.cache.kv_heads;
  Part* parts = static_cast<Part*>(p.workspace);
  float* sums = reinterpret_cast<float*>(parts + gridDim.x);
  constexpr int kSlot = kRows * (D + 2);
  Run r;
  Tile cur;
  if (!find_run<kRows, kThreads>(p, per, parts, r, cur)) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    return;
  }
  uint8_t* smem = dynamic + ((1024u - (smem_addr(dynamic) & 1023u)) & 1023u);
  const uint32_t raw_at = smem_addr(smem) + M::kRaw + threadIdx.x * 16;  // the thread's codes of values, 4 KB apart
  const uint32_t q_at = smem_addr(smem) + M::kQ, k_at = smem_addr(smem) + M::kK, v_at = smem_addr(smem) + M::kV;
  float* tok_a = reinterpret_cast<float*>(smem + M::kNums);
  float *tok_b = tok_a + kStep, *tok_l = tok_b + kStep, *tok_i = tok_l + kStep, *tok_v = tok_i + kStep;
  float* row_sum = tok_a + 2 * 5 * kStep;
  float *row_max = row_sum + kRows, *row_num = row_max + 2 * kRows;  // [half][row] each
  if (tid == 0) {
    mbar_init(&bar, 1);
    mbar_init(&keys_bar, kThreads / 32);
    mbar_init(&weights_bar, kThreads / 32);
    fence_mbar_init();
  }
  if (warp == 0) tmem_alloc(&tmem_slot, kTmemCols);
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  // Only now: a kernel that is set up early may take tensor memory before its wait, and this one's
  // blocks have theirs.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tmem = tmem_slot;
  uint32_t phase = 0, step_phase = 0;  // of products; of the barriers that complete once a step
  bool dead = false;
  auto wait_products = [&] {
    wait_phase(&bar, phase, dead, p);
    phase ^= 1;
  };
  // the warp's writes are done, for the products and the other warps
  auto arrive = [&](uint64_t* b) {
    tcgen05_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(b);
  };

  // this thread as a loader: half a token's codes (of a row's queries); as a row's: half its tokens
  const int tok = tid >> 1, part = tid & 1;
  const int row = (warp & 3) * 32 + lane, half = warp >> 2;
  const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
  const uint32_t t_s = tmem + lanes + half * 64, t_p = tmem + lanes + half * 32, t_o = tmem + lanes + kTmemO + half * (D / 2);
  const int page_mask = (1 << p.cache.shift) - 1;
  const float f = p.scale * 1.4426950408889634f;
  // where a loader's pieces go: at D = 128 its half's eight, begun with the fourth in the odd lanes, so
  // that the eight lanes of a store meet in no bank; at D = 64 four of the row's eight
  const uint32_t piece0 = H == 2 ? part * 4 : 0;
  auto piece = [&](uint32_t base, int c) {
    const uint32_t i = H == 2 ? (c ^ piece0) : (uint32_t)(part * 4 + c);
    return base + ((i ^ (uint32_t)(tok & 7)) << 4);
  };
  const uint32_t kq_row = (H == 2 ? part * (kRows * 128) : 0) + tok * 128;
  const uint32_t v_row = (tok >> 3) * (H * 1024) + (H == 2 ? part * 1024 : 0) + (tok & 7) * 128;
  auto put = [&](uint32_t at, const uint4& x) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w) : "memory");
  };

  auto get = [&](uint32_t at, uint32_t* x) {
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(at) : "memory");
  };
  auto copy16 = [&](uint32_t dst, const uint8_t* src, uint32_t size) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(size) : "memory");
  };

  long long at = r.start;
  for (;;) {
    const int end = cur.s.n * per - 1, row0 = cur.rt * kRows, rows = min(kRows, end + 1 - row0);
    auto sees = [&](int i) { return min(cur.s.kv, cur.s.last + min(row0 + i, end) / per + 1); };
    const int see = sees(row), see_least = sees(0), see_most = max(sees(kRows - 1), 0);
    const int s0 = max(cur.c0 - kTileCost, 0), s1 = min(max(cur.c1 - kTileCost, 0), (see_most + kStep - 1) / kStep);
    const int slot = at == r.start ? 0 : 1;
    float4* set_aside = reinterpret_cast<float4*>(sums + ((size_t)blockIdx.x * 2 + slot) * kSlot) + half * (D / 8) * kRows + row;
    const int* table = p.block_tables + (size_t)cur.b * p.max_blocks;

    // ---- the loads of a step ----
    int page = -1;
    bool there = false;
    uint32_t pair = 0;
    auto look = [&](int step) {
      const long long pos = (long long)step * kStep + tok;
      page = step < s1 && pos < see_most ? table[pos >> p.cache.shift] : -1;
    };
    // Codes of values wait in the thread's place, codes of keys in its own row of the operand, whose
    // products have completed; where nothing is there nothing is read.
    auto fetch = [&](int step) {
      there = (unsigned)page < (unsigned)p.cache.num_blocks;
      const long long at_row = there ? kv4_row(p.cache, page, cur.head, (step * kStep + tok) & page_mask) : 0;
      const long long at_code = at_row * (D / 2) + part * (D / 4);
      const uint32_t size = there ? 16 : 0;
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) {
        copy16(piece(k_at + kq_row, i), p.cache.k_codes + at_code + i * 16, size);
        copy16(raw_at + i * (kThreads * 16), p.cache.v_codes + at_code + i * 16, size);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      pair = there ? (part ? p.cache.v_scales : p.cache.k_scales)[at_row] : 0;
    };
    auto fetched = [&] { asm volatile("cp.async.wait_group 0;" ::: "memory"); };
    look(s0);

    // ---- queries: half a row a thread ----
    {
      const int i = min(row0 + tok, end), token = i / per;
      float sum = 0.f, odd = 0.f;
      const bool live = tok < rows && sees(tok) > 0;
      const long long src = (long long)(cur.s.first + token) * p.q_stride + (long long)(cur.head * per + i - token * per) * D +
                            part * (D / 2);
      uint4 x[D / 16];  // all under way before the first is looked at
#pragma unroll
      for (int c = 0; c < D / 16; ++c) {
        x[c] = make_uint4(0, 0, 0, 0);
        if (live) x[c] = load_bits8(static_cast<const uint16_t*>(p.q) + src + (H == 2 ? c ^ (part * 4) : c) * 8);
      }
#pragma unroll
      for (int c = 0; c < D / 16; ++c) {
        const uint32_t w[4] = {x[c].x, x[c].y, x[c].z, x[c].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float a = BF ? __uint_as_float(w[k] << 16) : half_lo(w[k]);
          const float b = BF ? __uint_as_float(w[k] & 0xFFFF0000u) : half_hi(w[k]);
          sum += a + b;
          odd = fmaf(a, 0.f, fmaf(b, 0.f, odd));  // NaN if one is not finite
        }
        put(piece(q_at + kq_row, c), x[c]);
      }
      sum += odd;
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      if (part == 0) row_sum[tok] = sum;
    }
    fetched();  // the last tile's last, of nothing
    fetch(s0);
    look(s0 + 1);

    float ref = -INFINITY, l = 0.f, off = 0.f, aside_ref = 0.f;
    bool fresh = true, pending = false, aside = false;  // O empty; products of O on their way; O in part in the slot
    int since = 0;
    for (int step = s0; step < s1; ++step) {
      // ---- keys, and the tokens' numbers ----
      const int turn = (int)step_phase * (5 * kStep);  // a warp may be a step ahead of another
      float m = 1.f;
      {
        const float scale = half_lo(pair), offset = half_hi(pair);
        if (part == 0) {
          tok_a[turn + tok] = f * scale;
          tok_b[turn + tok] = f * fmaf(8.f, scale, offset);
        } else {
          const float size = fabsf(scale), centre = fmaf(8.f, scale, offset);
          float lg = 0.f, inv = 1.f;
          if (!there) {
            lg = -INFINITY;  // weights of 0
            inv = m = 0.f;
          } else if (size == 0.f) {
            m = 0.f;
          } else if (!(size < INFINITY)) {
            inv = NAN;
          } else {
            lg = lg2(size);  // (normal in f32; an error of it is one of the weight, in both sums alike)
            inv = rcp(size);
            m = scale < 0.f ? -1.f : 1.f;
          }
          tok_l[turn + tok] = lg;
          tok_i[turn + tok] = inv;
          tok_v[turn + tok] = there ? centre * inv : 0.f;
        }
        m = __shfl_sync(0xffffffffu, m, lane | 1);
      }
      fetched();
      {
        uint32_t w[kWords];
#pragma unroll
        for (int i = 0; i < kWords / 4; ++i) get(piece(k_at + kq_row, i), w + 4 * i);
        // (the odd lanes' pieces are written from the fourth on)
#pragma unroll
        for (int c = 0; c < kWords; ++c) {
          const uint32_t x = kWords == 8 && part ? w[c ^ 4] : w[c];
          put(piece(k_at + kq_row, c), BF ? codes_bf16(x) : codes_f16(x, 0x3C003C00u, 0xE408E408u));
        }
      }
      fence_proxy_async_smem();
      if (pending) wait_products();
      if (since == kFlush) {
#pragma unroll 1
        for (int c = 0; c < D / 2; c += 16) {
          uint32_t o[16];
          tmem_load16(t_o + c, o);
          const float g = aside_ref == ref ? 1.f : ex2(aside_ref - ref);  // (neither has one yet: 1)
#pragma unroll
          for (int k = 0; k < 16; k += 4) {
            float4 x = make_float4(__uint_as_float(o[k]), __uint_as_float(o[k + 1]), __uint_as_float(o[k + 2]),
                                   __uint_as_float(o[k + 3]));
            float4* kept = set_aside + (c + k) / 4 * kRows;
            if (aside) add_scaled(x, *kept, g);
            *kept = x;
          }
        }
        aside_ref = ref;
        aside = fresh = true;
        since = 0;
      }
      arrive(&keys_bar);
      if (warp == 0) {
        wait_phase(&keys_bar, step_phase, dead, p);
        if (elect_one()) {
          constexpr uint32_t idesc = umma_idesc_f16(kRows, kStep) | (BF ? 1u << 7 | 1u << 10 : 0u);
          const uint64_t a = umma_smem_desc(q_at, 16, 1024, 2), b = umma_smem_desc(k_at, 16, 1024, 2);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint64_t d = ((kk >> 2) * (kRows * 128) + (kk & 3) * 32) >> 4;
            umma_f16(tmem, a + d, b + d, idesc, kk > 0);
          }
          umma_commit(&bar);
        }
        __syncwarp();
      }

      // ---- values, and the next step's loads ----
      {
        const uint32_t mm = m == 0.f ? 0u : (m < 0.f ? 0xBC00BC00u : 0x3C003C00u);
        const uint32_t shift = m == 0.f ? 0u : (m < 0.f ? 0x64086408u : 0xE408E408u);  // -1032 m
#pragma unroll
        for (int i = 0; i < kWords / 4; ++i) {
          uint32_t w[4];
          get(raw_at + (kWords == 8 ? i ^ part : i) * (kThreads * 16), w);
#pragma unroll
          for (int k = 0; k < 4; ++k) put(piece(v_at + v_row, 4 * i + k), codes_f16(w[k], mm, shift));
        }
        fence_proxy_async_smem();
      }

      // ---- scores ----
      wait_products();
      wait_phase(&keys_bar, step_phase, dead, p);  // (complete: the products were issued after it)
      uint32_t t[64];
      tmem_load64(t_s, t);
      const float q_sum = row_sum[row];
      const int pos0 = step * kStep + half * 64;  // below 2^31 - 1024
      const bool masked = (long long)step * kStep + kStep > see_least;
      float top = -INFINITY;
      auto score = [&](auto with_mask) {
        constexpr bool kMasked = decltype(with_mask)::value;
        const Pair q2 = pair_of(q_sum, q_sum);
#pragma unroll
        for (int j = 0; j < 64; j += 4) {
          Pair a[2], b[2], g[2];
          load_pairs(tok_a + turn + half * 64 + j, a);
          load_pairs(tok_b + turn + half * 64 + j, b);
          load_pairs(tok_l + turn + half * 64 + j, g);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int i = j + 2 * k;
            float2 x = values_of(fma2(a[k], pair_of(__uint_as_float(t[i]), __uint_as_float(t[i + 1])), fma2(b[k], q2, g[k])));
            if (kMasked && pos0 + i >= see) x.x = -INFINITY;
            if (kMasked && pos0 + i + 1 >= see) x.y = -INFINITY;
            t[i] = __float_as_uint(x.x);
            t[i + 1] = __float_as_uint(x.y);
            top = fmaxf(top, fmaxf(x.x, x.y));
          }
        }
      };
      if (masked)
        score(std::true_type{});
      else
        score(std::false_type{});
      // the two warps of these rows: both have read S, over which the weights go
      row_max[half * kRows + row] = top;
      tcgen05_fence_before();
      named_barrier(1 + (warp & 3), 64);
      tcgen05_fence_after();
      top = fmaxf(top, row_max[(1 - half) * kRows + row]);
      float fall = 1.f;
      if (top - ref > 15.f || (ref == -INFINITY && top > -INFINITY)) {
        fall = ex2(ref - (top - 10.f));
        ref = top - 10.f;
        l *= fall;
        off *= fall;
      }
      if (!fresh && __any_sync(0xffffffffu, fall != 1.f)) {
#pragma unroll 1
        for (int c = 0; c < D / 2; c += 16) {
          uint32_t o[16];
          tmem_load16(t_o + c, o);
#pragma unroll
          for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * fall);
          tmem_store16(t_o + c, o);
        }
      }

      fetch(step + 1);
      look(step + 2);

      // ---- weights ----
      auto weigh = [&](auto with_mask) {
        constexpr bool kMasked = decltype(with_mask)::value;
        const float r0 = ref == -INFINITY ? 0.f : -ref;
        const Pair r2 = pair_of(r0, r0);
        Pair l2 = pair_of(l, 0.f), off2 = pair_of(off, 0.f);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t hi[16], lo[16];
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            Pair inv[2], v[2];
            load_pairs(tok_i + turn + half * 64 + c * 32 + j, inv);
            load_pairs(tok_v + turn + half * 64 + c * 32 + j, v);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const int i = c * 32 + j + 2 * k;
              float2 w = values_of(add2(pair_of(__uint_as_float(t[i]), __uint_as_float(t[i + 1])), r2));
              w.x = ex2(w.x);
              w.y = ex2(w.y);
              const Pair w2 = pair_of(w.x, w.y);
              if (kMasked) {  // what the numbers of hidden tokens are does not matter
                const bool hide_x = pos0 + i >= see, hide_y = pos0 + i + 1 >= see;
                float2 a = values_of(inv[k]), b = values_of(v[k]);
                inv[k] = pair_of(hide_x ? 0.f : a.x, hide_y ? 0.f : a.y);
                v[k] = pair_of(hide_x ? 0.f : b.x, hide_y ? 0.f : b.y);
              }
              l2 = fma2(w2, inv[k], l2);
              off2 = fma2(w2, v[k], off2);
              const uint32_t h = pack_f16(w.x, w.y);
              const float2 rest = values_of(add2(w2, pair_of(-half_lo(h), -half_hi(h))));
              hi[j / 2 + k] = h;
              lo[j / 2 + k] = pack_f16(rest.x, rest.y);
            }
          }
          tmem_store16(t_p + c * 16, hi);
          tmem_store16(t_p + kTmemLow + c * 16, lo);
        }
        const float2 a = values_of(l2), b = values_of(off2);
        l = a.x + a.y;
        off = b.x + b.y;
      };
      if (masked)
        weigh(std::true_type{});
      else
        weigh(std::false_type{});
      tmem_st_wait();
      arrive(&weights_bar);
      if (warp == 0) {
        wait_phase(&weights_bar, step_phase, dead, p);
        if (elect_one()) {
          constexpr uint32_t idesc = umma_idesc_f16(kRows, D) | 1u << 16;  // B by rows of the k dimension
          const uint64_t b = umma_smem_desc(v_at, 1024, H * 1024, 2);
#pragma unroll
          for (int kk = 0; kk < kStep / 16; ++kk) {
            const uint64_t d = b + (uint64_t)(kk * (H * 2048) >> 4);
            umma_f16_ts(tmem + kTmemO, tmem + 8 * kk, d, idesc, !fresh || kk > 0);
            umma_f16_ts(tmem + kTmemO, tmem + kTmemLow + 8 * kk, d, idesc, 1);
          }
          umma_commit(&bar);
        }
        __syncwarp();
      }
      step_phase ^= 1;
      fresh = false;
      pending = true;
      ++since;
    }
    if (pending) wait_products();

    // ---- the tile's end ----
    row_max[half * kRows + row] = l;
    row_num[half * kRows + row] = off;
    __syncthreads();
    l += row_max[(1 - half) * kRows + row];
    off += row_num[(1 - half) * kRows + row];
    const bool whole = cur.c0 == 0 && cur.c1 == cur.s.steps;
    const float g = aside_ref == ref ? 1.f : ex2(aside_ref - ref);  // (neither has one yet: 1)
    const int i = min(row0 + row, end), token = i / per;
    const long long o_at = (long long)(cur.s.first + token) * p.o_stride + (long long)(cur.head * per + i - token * per) * D +
                           half * (D / 2);
    const float over = l == 0.f ? 0.f : 1.f / l;
#pragma unroll 1
    for (int c = 0; c < D / 2; c += 16) {
      uint32_t o[16];
      if (!fresh)
        tmem_load16(t_o + c, o);
      else
#pragma unroll
        for (int k = 0; k < 16; ++k) o[k] = 0;
      float4 x[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        x[k] = make_float4(__uint_as_float(o[4 * k]) + off, __uint_as_float(o[4 * k + 1]) + off,
                           __uint_as_float(o[4 * k + 2]) + off, __uint_as_float(o[4 * k + 3]) + off);
        float4* kept = set_aside + (c / 4 + k) * kRows;
        if (aside) add_scaled(x[k], *kept, g);
        if (!whole) *kept = x[k];
      }
      if (whole && row < rows) {
        if (l == 0.f) x[0] = x[1] = x[2] = x[3] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < 4; k += 2) {
          const uint4 y = make_uint4(pack_out<BF>(x[k].x * over, x[k].y * over), pack_out<BF>(x[k].z * over, x[k].w * over),
                                     pack_out<BF>(x[k + 1].x * over, x[k + 1].y * over),
                                     pack_out<BF>(x[k + 1].z * over, x[k + 1].w * over));
          store_bits8(static_cast<uint16_t*>(p.o) + o_at + c + 4 * k, y);
        }
      }
    }
    if (!whole && half == 0) {
      float* num = sums + ((size_t)blockIdx.x * 2 + slot) * kSlot + kRows * D + 2 * row;
      num[0] = ref;
      num[1] = l;
    }
    if (!whole && cur.c0 == 0 && tid == 0)
      parts[blockIdx.x] = Part{cur.s.first, rows, cur.head, (int)((at + cur.s.steps - 1) / r.length - blockIdx.x + 1), row0,
                               slot, 0, 0};
    at += cur.c1 - cur.c0;
    if (at >= r.stop) break;
    next_tile<kRows>(p, per, at, r.stop, cur);
    tcgen05_fence_before();
    __syncthreads();  // the rows' numbers have been read
  }
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 0) tmem_dealloc(tmem, kTmemCols);
}

// Joins the parts of the tile that begins in the run of CTA blockIdx.x, kJoinDims dimensions of it: a
// thread a row, four parts under way at a time.
constexpr int kJoinDims = 16, kJoinParts = 4;
template <int D, bool BF>
__global__ void __launch_bounds__(kRows) kv4_prompt_join_kernel(Kv4AttentionParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const Part* parts = static_cast<const Part*>(p.workspace);
  const float* sums = reinterpret_cast<const float*>(parts + gridDim.x);
  constexpr int kSlot = kRows * (D + 2), V = kJoinDims / 4;
  const Part part = parts[blockIdx.x];
  const int row = threadIdx.x;
  if (part.count == 0 || row >= part.rows) return;
  const int d0 = blockIdx.y * kJoinDims;
  float top = -INFINITY, sum = 0.f;
  float4 v[V];
#pragma unroll
  for (int k = 0; k < V; ++k) v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = 0; i0 < part.count; i0 += kJoinParts) {
    float2 num[kJoinParts];
    float4 x[kJoinParts][V];
    float now = top;
#pragma unroll
    for (int u = 0; u < kJoinParts; ++u) {
      const int i = min(i0 + u, part.count - 1);  // one that counts, read again
      const float* s = sums + ((size_t)(blockIdx.x + i) * 2 + (i == 0 ? part.slot : 0)) * kSlot;
      num[u] = *reinterpret_cast<const float2*>(s + kRows * D + 2 * row);
#pragma unroll
      for (int k = 0; k < V; ++k) x[u][k] = reinterpret_cast<const float4*>(s)[(d0 / 4 + k) * kRows + row];
      now = fmaxf(now, num[u].x);
    }
    const float f = top == now ? 1.f : ex2(top - now);  // (no reference yet: sums of 0, or of NaN)
    top = now;
    sum *= f;
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = make_float4(v[k].x * f, v[k].y * f, v[k].z * f, v[k].w * f);
#pragma unroll
    for (int u = 0; u < kJoinParts; ++u) {
      if (i0 + u >= part.count) break;
      const float g = num[u].x == now ? 1.f : ex2(num[u].x - now);
      sum = fmaf(num[u].y, g, sum);
#pragma unroll
      for (int k = 0; k < V; ++k) add_scaled(v[k], x[u][k], g);
    }
  }
  const int per = p.q_heads / p.cache.kv_heads, q = part.row0 + row;
  const long long at = (long long)(part.token + q / per) * p.o_stride + (long long)(part.head * per + q % per) * D + d0;
  const float over = sum == 0.f ? 0.f : 1.f / sum;
  if (sum == 0.f) {
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
#pragma unroll
  for (int k = 0; k < V; k += 2)
    store_bits8(static_cast<uint16_t*>(p.o) + at + 4 * k,
                make_uint4(pack_out<BF>(v[k].x * over, v[k].y * over), pack_out<BF>(v[k].z * over, v[k].w * over),
                           pack_out<BF>(v[k + 1].x * over, v[k + 1].y * over),
                           pack_out<BF>(v[k + 1].z * over, v[k + 1].w * over)));
}

template <int D, bool BF>
cudaError_t launch(Kv4AttentionParams p, int sm_count, cudaStream_t st) {
  constexpr int smem = PromptSmem<D>::kBytes, kMaxDevices = 64;
  static std::atomic<unsigned> asked[kMaxDevices];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const unsigned gen = attr_generation(dev) + 1;
  if (dev >= kMaxDevices || asked[dev].load(std::memory_order_acquire) != gen) {
    e = cudaFuncSetAttribute(kv4_prompt_kernel<D, BF>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    if (dev < kMaxDevices) asked[dev].store(gen, std::memory_order_release);
  }
  const int ctas = sm_count * kCtasPerSm;
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
  e = cudaLaunchKernelEx(&cfg, kv4_prompt_kernel<D, BF>, p);
  if (e != cudaSuccess) return e;
  cfg.dynamicSmemBytes = 0;
  cfg.gridDim = dim3((unsigned)ctas, D / kJoinDims);
  cfg.blockDim = dim3(kRows);
  return cudaLaunchKernelEx(&cfg, kv4_prompt_join_kernel<D, BF>, p);
}

}  // namespace

// Queries of 16 bits (one product with them is exact), one group a head, and on the mean enough rows a
// sequence: against tiles of eight rows, 16 x 2000 positions with 32 rows a head take 64 us instead of
// 53, with 48 65 instead of 73, with 128 70 instead of 168; 60000 positions 110 and 75, 111 and 106, 114
// and 255.  A step is long, so little work in all wants more rows (one sequence of 3000, by the table's
// reach: 48 rows 29 and 19 us, 128 rows 32 and 28, 256 rows 33 and 40).
bool kv4_prompt_takes(const Kv4AttentionParams& p, int dtype) {
  if (dtype == kTypeF32 || p.cache.head_dim > 128 || p.cache.group != p.cache.head_dim) return false;
  const long long rows = (long long)p.tokens * (p.q_heads / p.cache.kv_heads);
  const long long tiles = (rows / kRows + p.batch) * p.cache.kv_heads;
  const long long steps = (((long long)p.max_blocks << p.cache.shift) + kStep - 1) / kStep + kTileCost;
  return rows >= 160ll * p.batch || (rows >= 48ll * p.batch && tiles * steps >= 600);
}

size_t kv4_prompt_workspace(int head_dim, int sm_count) {
  return head_dim > 128 ? 0 : attention_workspace(sm_count * kCtasPerSm, kRows, head_dim);
}

cudaError_t launch_kv4_prompt(Kv4AttentionParams p, int dtype, int sm_count, cudaStream_t st) {
  if (p.cache.head_dim == 64)
    return dtype == kTypeBF16 ? launch<64, true>(p, sm_count, st) : launch<64, false>(p, sm_count, st);
  return dtype == kTypeBF16 ? launch<128, true>(p, sm_count, st) : launch<128, false>(p, sm_count, st);
}

}  // namespace tk
