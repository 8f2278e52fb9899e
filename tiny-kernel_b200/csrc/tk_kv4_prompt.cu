// tk_kv4_prompt.cu -- attention over the 4-bit cache for many query rows a key head: prompts and
// their chunks.
//
// The mathematics is that of tk_kv4_attention.cu, with the products on tcgen05: a tile is 128 rows (query
// token, head of the group) against 64 or 128 tokens a step.  For each group of dimensions
//   S = Q (c - 8)^T    Q as it is (f16 or bf16; f32 as two f16, 22 bits of the row's largest), the codes exact
//   t = sum over groups of (a S + b sum(q)) + e,   a = f s_k, b = f (m_k + 8 s_k), f = scale log2 e
//   w = 2^(t - r + log2 |s_v| - e),  O += w sign(s_v) (c - 8),  off += w (m_v + 8 s_v) / |s_v|
// with e the largest log2 |s_v| of the token's groups; l += w / |s_v| of the first; o = (O + off) / l.  So
// a weight comes out of the exponential with its scale in it, ready for the second product; it is split
// into two f16 (22 bits), two products into one accumulator.  s_v = 0 counts as 1 with values of 0.  A
// row's reference r keeps the weights below 2^15; when one would pass, r is moved so that the largest is
// 2^10, and the sums are rescaled, which is rare.
//
// One CTA is 256 threads, two a row: half of a step's tokens each, and half of the dimensions of O.
// Tensor memory: S, over which the weights lie as f16 pairs once all of S has been read, and O.  A step
// is one chain (unpack keys, S, weights, O), so two CTAs live on an SM (one at 256 dimensions), one
// computing while the other's products run.  Warps wait for products, the two of a row for each other,
// and one, which issues the products, for all.  The next step's codes travel meanwhile: those of keys
// into the operand's own rows, whose products have completed.
//   The tensor core's sums round toward zero: O is set aside into the CTA's slot of the workspace every
// 2048 tokens (256 of f32 queries, whose outputs would show it), and l and off with it, each a sum of the
// steps' sums until then.  Those additions are compensated: what one drops begins the next interval, O's in
// tensor memory.  So an error does not grow with the length: equal tokens and weights, f32, 2048 positions in
// one CTA 0.3e-6 of the result, 131072 0.3e-6 (as plain running sums 8e-6 and 325e-6).  S has eight products a
// row; of f32 queries the low part's eight go first, whose sum has little to drop.  2 x 256 tokens over 1500 to
// 4000 positions, f32: 1.36e-6 of the result, 1.44e-6 in f32 torch operations (the high part first, every 512
// tokens: 2.84e-6 and 149 us instead of 157; the low part first alone 1.78e-6); the exact integers of smaller tiles give 0.4
// to 1.2e-6.
//
// What bounds it (B200; those 2 x 256 tokens, 40 + 8 heads of 128, bf16): 109 us, 298 TFLOP/s with one
// product each (the second part of the weights is a third one); tiles of eight rows on mma.sync take 301.
// f32: 157 and 301.  Instruction issue and its latencies: 1400 instructions a warp and step at 0.47 a
// cycle and scheduler, four warps a scheduler (128 registers, most of them scores), tensor pipe 24 %
// busy.  When a call took 118 us, numbers of tokens for eight instead of four columns at a time made it
// 125 (spilled); when it took 112, one f16 part of a weight instead of two 102, with 11 bits.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "tk_internal.h"
#include "tk_kv4_attention.cuh"
#include "tk_ptx.cuh"

namespace tk {
namespace {

constexpr int kRows = kManyRows, kThreads = 256;
constexpr unsigned kErrPromptWait = 64u;  // a product, or a warp, of a prompt never completed

// Waits, a warp together, for the phase of `bar`; gives up, for good, after timeout_ns.
__device__ __forceinline__ void wait_phase(uint64_t* bar, uint32_t phase, bool& dead, const Kv4AttentionParams& p) {
  if (!dead && !mbar_try_wait(bar, phase)) {
    const uint64_t t0 = global_timer_ns();
    while (!mbar_try_wait(bar, phase))
      if (global_timer_ns() - t0 > p.timeout_ns) {
        atomicOr(p.err, kErrPromptWait);
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
// 64, 32 or 16 consecutive columns of the warp's 32 lanes, complete on return.
__device__ __forceinline__ void tmem_load(uint32_t at, uint32_t (&r)[64]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, %34, %35, "
      "%36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, "
      "%57, %58, %59, %60, %61, %62, %63}, [%64];\n\ttcgen05.wait::ld.sync.aligned;"
      : TK_R16(r, 0), TK_R16(r, 16), TK_R16(r, 32), TK_R16(r, 48)
      : "r"(at)
      : "memory");
}
__device__ __forceinline__ void tmem_load(uint32_t at, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : TK_R16(r, 0), TK_R16(r, 16)
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
__device__ __forceinline__ void load_eight(const float* src, bool live, float (&v)[8]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = 0.f;
  if (!live) return;
  if (reinterpret_cast<uintptr_t>(src) % 16 == 0) {
    const float4 a = reinterpret_cast<const float4*>(src)[0], b = reinterpret_cast<const float4*>(src)[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = src[k];
  }
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
// N * 4 values of a row over their sum, l (none: zeros).
template <int TYPE, int N>
__device__ __forceinline__ void store_rows(void* o, long long at, float4 (&x)[N], float l, float over) {
  if (l == 0.f) {
#pragma unroll
    for (int k = 0; k < N; ++k) x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  if constexpr (TYPE == kTypeF32) {
    float* dst = static_cast<float*>(o) + at;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const float4 y = make_float4(x[k].x * over, x[k].y * over, x[k].z * over, x[k].w * over);
      if (reinterpret_cast<uintptr_t>(dst) % 16 == 0)
        reinterpret_cast<float4*>(dst)[k] = y;
      else
        dst[4 * k] = y.x, dst[4 * k + 1] = y.y, dst[4 * k + 2] = y.z, dst[4 * k + 3] = y.w;
    }
  } else {
    constexpr bool BF = TYPE == kTypeBF16;
#pragma unroll
    for (int k = 0; k < N; k += 2)
      store_bits8(static_cast<uint16_t*>(o) + at + 4 * k,
                  make_uint4(pack_out<BF>(x[k].x * over, x[k].y * over), pack_out<BF>(x[k].z * over, x[k].w * over),
                             pack_out<BF>(x[k + 1].x * over, x[k + 1].y * over),
                             pack_out<BF>(x[k + 1].z * over, x[k + 1].w * over)));
  }
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
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair y;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(y.x) : "l"(a.x), "l"(b.x));
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

// What a head's size, its groups and the queries' type make of the kernel.
template <int D, int G, int TYPE>
struct Form {
  static constexpr bool kF32 = TYPE == kTypeF32, kBF16 = TYPE == kTypeBF16;
  static constexpr int kGroups = D / G, kHalves = D / 64;  // operands lie in halves of a head of 128, 128 bytes a row
  // Tokens of a step: as many as tensor memory (a product a group) and shared memory (f32 queries are
  // two parts) leave room for.
  static constexpr int kTokens = kGroups == 1 && !(kF32 && D == 128) ? 128 : 64;
  static constexpr int kCtas = D == 256 ? 1 : 2;  // of an SM
  static constexpr uint32_t kTmem = 512 / kCtas, kTmemO = kTmem / 2;
  static constexpr int kFlush = (kF32 ? 256 : 2048) / kTokens;
  static constexpr int kLoaders = kThreads / kTokens;      // threads of a token
  static constexpr int kWords = D / kLoaders / 8;          // of codes, eight each, a thread
  // per token and group a, b, log2 |s_v| less the groups' largest, (m_v + 8 s_v) / |s_v|; per token the
  // largest, and 1 / |s_v| of the first group
  static constexpr int kNumbers = kGroups == 1 ? 5 : 4 * kGroups + 2;
  static_assert(kGroups * kTokens <= (int)kTmemO && D <= (int)kTmemO, "tensor memory");
  // Shared memory: queries [part][half][row], keys [half][token], values by eights of tokens [token / 8]
  // [half][token % 8], their 16-byte pieces turned by the row's number; codes of values as they come;
  // numbers of the tokens, twice; per row a group's sum(q), what undoes f32 queries' factor, and two
  // halves' numbers.
  static constexpr int kQPart = kRows * D * 2, kOperand = kTokens * D * 2;
  static constexpr int kQ = 0, kK = (kF32 ? 2 : 1) * kQPart, kV = kK + kOperand, kRaw = kV + kOperand;
  static constexpr int kNums = kRaw + kTokens * D / 2;
  static constexpr int kRowNums = kGroups + (kF32 ? 1 : 0) + 2 + 2 * kGroups;
  static constexpr int kBytes = kNums + (2 * kNumbers * kTokens + kRowNums * kRows) * 4 + 1024;
};

template <int D, int G, int TYPE>
__global__ void __launch_bounds__(kThreads, Form<D, G, TYPE>::kCtas) kv4_prompt_kernel(Kv4AttentionParams p) {
  using M = Form<D, G, TYPE>;
  constexpr int NG = M::kGroups, H = M::kHalves, TOK = M::kTokens, T2 = TOK / 2, L = M::kLoaders, W = M::kWords;
  constexpr bool F32 = M::kF32, BF = M::kBF16;
  constexpr uint32_t kO = M::kTmemO;
  extern __shared__ uint8_t dynamic[];
  __shared__ uint64_t bar, keys_bar, weights_bar;  // products complete; all warps' keys, weights written
  __shared__ uint64_t all_bar;                     // (after a wait gave up) all products complete
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
  const uint32_t q_at = smem_addr(smem) + M::kQ, k_at = smem_addr(smem) + M::kK, v_at = smem_addr(smem) + M::kV;
  const uint32_t raw_at = smem_addr(smem) + M::kRaw + threadIdx.x * 16;  // the thread's codes of values, 4 KB apart
  // [number][token], twice; [number][row]
  float* tok_a = reinterpret_cast<float*>(smem + M::kNums);
  float *tok_b = tok_a + NG * TOK, *tok_v = tok_b + NG * TOK, *tok_l = tok_v + NG * TOK, *tok_i = tok_l + TOK;
  float* tok_d = tok_i + TOK;  // (of several groups)
  float* row_sum = tok_a + 2 * M::kNumbers * TOK;
  float *row_max = row_sum + NG * kRows, *row_off = row_max + 2 * kRows, *row_undo = row_off + 2 * NG * kRows;
  if (tid == 0) {
    mbar_init(&bar, 1);
    mbar_init(&all_bar, 1);
    mbar_init(&keys_bar, kThreads / 32);
    mbar_init(&weights_bar, kThreads / 32);
    fence_mbar_init();
  }
  if (warp == 0) tmem_alloc(&tmem_slot, M::kTmem);
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

  // this thread as a loader: a half or a quarter of a token's codes; as a row's: half of its tokens
  const int tok = tid / L, part = tid % L;
  const int row = (warp & 3) * 32 + lane, half = warp >> 2;
  const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
  const uint32_t t_s = tmem + lanes + half * T2, t_p = tmem + lanes + half * (T2 / 2), t_o = tmem + lanes + kO + half * (D / 2);
  const int page_mask = (1 << p.cache.shift) - 1;
  const float f = p.scale * 1.4426950408889634f;
  // Where a loader's pieces go.  Threads with eight begin with the fourth in the odd lanes, whose rows
  // lie in the banks of the even ones'.
  const uint32_t second = W == 8 ? part & 1 : 0;
  auto piece_k = [&](int i) {
    const uint32_t k = part * W + i;
    return k_at + (k >> 3) * (TOK * 128) + tok * 128 + (((k & 7) ^ (uint32_t)(tok & 7)) << 4);
  };
  auto piece_v = [&](int i) {
    const uint32_t k = part * W + i;
    return v_at + (tok >> 3) * (H * 1024) + (k >> 3) * 1024 + (tok & 7) * 128 + (((k & 7) ^ (uint32_t)(tok & 7)) << 4);
  };
  auto put = [&](uint32_t at, const uint4& x) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w) : "memory");
  };
  auto get = [&](uint32_t at, uint32_t* x) {
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(at) : "memory");
  };
  auto copy16 = [&](uint32_t dst, const uint8_t* src, uint32_t size) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(size) : "memory");
  };
  // The token's numbers: of its groups' keys and values, one or both of a group a thread; the group
  // that the thread's dimensions lie in, and who has its numbers.
  const int group = NG == 4 ? part : part >> 1;
  const bool has_k = NG == 4 || (part % 2 == 0 && group < NG), has_v = NG == 4 || (part % 2 == 1 && group < NG);
  const int v_lane = (lane & ~(L - 1)) + (NG == 4 ? part : NG == 2 ? (part | 1) : 1);

  long long at = r.start;
  for (;;) {
    const int end = cur.s.n * per - 1, row0 = cur.rt * kRows, rows = min(kRows, end + 1 - row0);
    auto sees = [&](int i) { return min(cur.s.kv, cur.s.last + min(row0 + i, end) / per + 1); };
    const int see = sees(row), see_least = sees(0), see_most = max(sees(kRows - 1), 0);
    constexpr int kParts = kStep / TOK;  // steps here of one of the partition's
    const int s0 = max(cur.c0 - kTileCost, 0) * kParts;
    const int s1 = min(max(cur.c1 - kTileCost, 0) * kParts, (see_most + TOK - 1) / TOK);
    const int slot = at == r.start ? 0 : 1;
    // where the half's dimensions c .. c + 3 are set aside: (half * D / 8 + c / 4) * kRows + row
    float4* set_aside = reinterpret_cast<float4*>(sums + ((size_t)blockIdx.x * 2 + slot) * kSlot) + half * (D / 8) * kRows + row;
    // l goes where the row's reference and l are left at the tile's end, off where its parts meet there
    auto aside_l = [&]() -> float& { return sums[((size_t)blockIdx.x * 2 + slot) * kSlot + kRows * D + 2 * row + half]; };
    auto aside_off = [&](int y) -> float& { return row_off[(2 * y + half) * kRows + row]; };
    const int* table = p.block_tables + (size_t)cur.b * p.max_blocks;

    // ---- the loads of a step ----
    int page = -1;
    bool there = false;
    uint32_t k_pair = 0, v_pair = 0;
    auto look = [&](int step) {
      const long long pos = (long long)step * TOK + tok;
      page = step < s1 && pos < see_most ? table[pos >> p.cache.shift] : -1;
    };
    // Codes of values wait in the thread's place, codes of keys in its own row of the operand, whose
    // products have completed; where nothing is there nothing is read.
    auto fetch = [&](int step) {
      there = (unsigned)page < (unsigned)p.cache.num_blocks;
      const long long at_row = there ? kv4_row(p.cache, page, cur.head, (step * TOK + tok) & page_mask) : 0;
      const long long at_code = at_row * (D / 2) + part * (W * 4);
      const uint32_t size = there ? 16 : 0;
#pragma unroll
      for (int i = 0; i < W / 4; ++i) {
        copy16(piece_k(i), p.cache.k_codes + at_code + i * 16, size);
        copy16(raw_at + i * (kThreads * 16), p.cache.v_codes + at_code + i * 16, size);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      if (NG == 4) {
        k_pair = there ? p.cache.k_scales[at_row * NG + group] : 0;
        v_pair = there ? p.cache.v_scales[at_row * NG + group] : 0;
      } else {  // one of them
        k_pair = there && group < NG ? (has_v ? p.cache.v_scales : p.cache.k_scales)[at_row * NG + group] : 0;
        v_pair = k_pair;
      }
    };
    auto fetched = [&] { asm volatile("cp.async.wait_group 0;" ::: "memory"); };
    look(s0);

    // ---- queries: half a row a thread ----
    {
      const int q_row = tid >> 1, q_part = tid & 1;
      const int i = min(row0 + q_row, end), token = i / per;
      const bool live = q_row < rows && sees(q_row) > 0;
      const long long src = (long long)(cur.s.first + token) * p.q_stride + (long long)(cur.head * per + i - token * per) * D +
                            q_part * (D / 2);
      auto piece_q = [&](int i8, int which) {
        const uint32_t k = q_part * (D / 16) + i8;
        return q_at + which * M::kQPart + (k >> 3) * (kRows * 128) + q_row * 128 + (((k & 7) ^ (uint32_t)(q_row & 7)) << 4);
      };
      constexpr int kBlock = 8 < D / 16 ? 8 : D / 16;  // pieces under way at a time
      constexpr int kOwn = NG < 2 ? 1 : NG / 2;        // groups of half a row
      float sum[kOwn], odd = 0.f;
#pragma unroll
      for (int k = 0; k < kOwn; ++k) sum[k] = 0.f;
      const uint32_t second_q = D >= 128 ? q_part * 4 : 0;  // as above
      if constexpr (!F32) {
#pragma unroll
        for (int c0 = 0; c0 < D / 16; c0 += kBlock) {
          uint4 x[kBlock];  // all under way before the first is looked at
#pragma unroll
          for (int c = 0; c < kBlock; ++c) {
            x[c] = make_uint4(0, 0, 0, 0);
            if (live) x[c] = load_bits8(static_cast<const uint16_t*>(p.q) + src + (c0 + (c ^ second_q)) * 8);
          }
#pragma unroll
          for (int c = 0; c < kBlock; ++c) {
            const uint32_t w[4] = {x[c].x, x[c].y, x[c].z, x[c].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float a = BF ? __uint_as_float(w[k] << 16) : half_lo(w[k]);
              const float b = BF ? __uint_as_float(w[k] & 0xFFFF0000u) : half_hi(w[k]);
              sum[c0 * 8 / G % kOwn] += a + b;  // (a block lies in one group)
              odd = fmaf(a, 0.f, fmaf(b, 0.f, odd));  // NaN if one is not finite
            }
            put(piece_q(c0 + (c ^ second_q), 0), x[c]);
          }
        }
      } else {
        // the largest becomes 2^14 .. 2^15; two f16 hold 22 bits of it and of what is 2^-17 of it
        float top = 0.f;
#pragma unroll
        for (int c0 = 0; c0 < D / 16; c0 += 4) {
          float v[4][8];
#pragma unroll
          for (int c = 0; c < 4; ++c) load_eight(static_cast<const float*>(p.q) + src + (c0 + c) * 8, live, v[c]);
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              top = fmaxf(top, fabsf(v[c][k]));
              odd = fmaf(v[c][k], 0.f, odd);
              sum[c0 * 8 / G % kOwn] += v[c][k];
            }
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        const int e = top > 0.f && top < INFINITY ? min(14 - ilogbf(top), 120) : 0;
        const float norm = ldexpf(1.f, e);
        if (q_part == 0) row_undo[q_row] = ldexpf(1.f, -e);
#pragma unroll
        for (int c0 = 0; c0 < D / 16; c0 += 4) {
          float v[4][8];
#pragma unroll
          for (int c = 0; c < 4; ++c) load_eight(static_cast<const float*>(p.q) + src + (c0 + c) * 8, live, v[c]);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) split_f16(v[c][2 * k] * norm, v[c][2 * k + 1] * norm, hi[k], lo[k]);
            put(piece_q(c0 + c, 0), make_uint4(hi[0], hi[1], hi[2], hi[3]));
            put(piece_q(c0 + c, 1), make_uint4(lo[0], lo[1], lo[2], lo[3]));
          }
        }
      }
      odd += __shfl_xor_sync(0xffffffffu, odd, 1);
      if constexpr (NG == 1) {
        sum[0] += __shfl_xor_sync(0xffffffffu, sum[0], 1);
        if (q_part == 0) row_sum[q_row] = sum[0] + odd;
      } else {
#pragma unroll
        for (int k = 0; k < kOwn; ++k) row_sum[(q_part * kOwn + k) * kRows + q_row] = sum[k] + odd;
      }
    }
    fetched();  // the last tile's last, of nothing
    fetch(s0);
    look(s0 + 1);

    float ref = -INFINITY, l = 0.f, off[NG], aside_ref = 0.f;
#pragma unroll
    for (int g = 0; g < NG; ++g) off[g] = 0.f;
    bool fresh = true, pending = false, aside = false;  // O empty; products of O on their way; O in part in the slot
    int since = 0;
    for (int step = s0; step < s1; ++step) {
      // ---- keys, and the tokens' numbers ----
      const int turn = (int)step_phase * (M::kNumbers * TOK);  // a warp may be a step ahead of another
      float m = 1.f;
      {
        if (has_k) {
          const float scale = half_lo(k_pair), offset = half_hi(k_pair);
          tok_a[turn + group * TOK + tok] = f * scale;
          tok_b[turn + group * TOK + tok] = f * fmaf(8.f, scale, offset);
        }
        float lg = -INFINITY;  // weights of 0
        if (has_v) {
          const float scale = half_lo(v_pair), size = fabsf(scale), centre = fmaf(8.f, scale, half_hi(v_pair));
          float inv = 1.f, v = centre;
          if (!there) {
            inv = m = v = 0.f;
          } else if (size == 0.f) {
            lg = m = 0.f;
          } else if (!(size < INFINITY)) {
            lg = 0.f;
            v = NAN;
          } else {
            lg = lg2(size);  // (normal in f32; an error of it is one of the weight, in both sums alike)
            inv = rcp(size);
            v = centre * inv;
            m = scale < 0.f ? -1.f : 1.f;
          }
          if (group == 0) tok_i[turn + tok] = inv;
          tok_v[turn + group * TOK + tok] = v;
        }
        float most = lg;
        if constexpr (NG > 1) {  // of the groups
          most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
          most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
          if (has_v) tok_d[turn + group * TOK + tok] = there ? lg - most : 0.f;
        }
        if (has_v && group == 0) tok_l[turn + tok] = most;
        if (NG != 4) m = __shfl_sync(0xffffffffu, m, v_lane);
      }
      fetched();
      {
        uint32_t w[W];
#pragma unroll
        for (int i = 0; i < W / 4; ++i) get(piece_k(i ^ second), w + 4 * i);
#pragma unroll
        for (int c = 0; c < W; ++c)
          put(piece_k(c ^ (second * 4)), BF ? codes_bf16(w[c]) : codes_f16(w[c], 0x3C003C00u, 0xE408E408u));
      }
      fence_proxy_async_smem();
      if (pending) wait_products();
      if (since == M::kFlush) {
        // the sums so far, of another reference perhaps; what rounding drops of them begins the next ones
        const float g = aside_ref == ref ? 1.f : ex2(aside_ref - ref);  // (neither has one yet: 1)
        l = keep(aside, aside_l(), g, l);
#pragma unroll
        for (int y = 0; y < NG; ++y) off[y] = keep(aside, aside_off(y), g, off[y]);
#pragma unroll 1
        for (int c = 0; c < D / 2; c += 16) {
          uint32_t o[16];
          tmem_load16(t_o + c, o);
#pragma unroll
          for (int k = 0; k < 16; k += 4) {
            float4* kept = set_aside + (c + k) / 4 * kRows;
            float4 x = *kept;
            o[k] = __float_as_uint(keep(aside, x.x, g, __uint_as_float(o[k])));
            o[k + 1] = __float_as_uint(keep(aside, x.y, g, __uint_as_float(o[k + 1])));
            o[k + 2] = __float_as_uint(keep(aside, x.z, g, __uint_as_float(o[k + 2])));
            o[k + 3] = __float_as_uint(keep(aside, x.w, g, __uint_as_float(o[k + 3])));
            *kept = x;
          }
          tmem_store16(t_o + c, o);
        }
        tmem_st_wait();
        aside_ref = ref;
        aside = true;
        since = 0;
      }
      arrive(&keys_bar);
      if (warp == 0) {
        wait_phase(&keys_bar, step_phase, dead, p);
        if (elect_one()) {
          constexpr uint32_t idesc = umma_idesc_f16(kRows, TOK) | (BF ? 1u << 7 | 1u << 10 : 0u);
          const uint64_t a = umma_smem_desc(q_at, 16, 1024, 2), b = umma_smem_desc(k_at, 16, 1024, 2);
#pragma unroll
          for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int q = F32 ? 1 : 0; q >= 0; --q)  // the low part first
#pragma unroll
              for (int i = 0; i < G / 16; ++i) {
                const int kk = g * (G / 16) + i;
                umma_f16(tmem + g * TOK, a + ((q * M::kQPart + (kk >> 2) * (kRows * 128) + (kk & 3) * 32) >> 4),
                         b + (((kk >> 2) * (TOK * 128) + (kk & 3) * 32) >> 4), idesc, q < (F32 ? 1 : 0) || i > 0);
              }
          umma_commit(&bar);
        }
        __syncwarp();
      }

      // ---- values ----
      {
        const uint32_t mm = m == 0.f ? 0u : (m < 0.f ? 0xBC00BC00u : 0x3C003C00u);
        const uint32_t shift = m == 0.f ? 0u : (m < 0.f ? 0x64086408u : 0xE408E408u);  // -1032 m
#pragma unroll
        for (int i = 0; i < W / 4; ++i) {
          uint32_t w[4];
          get(raw_at + (i ^ second) * (kThreads * 16), w);
#pragma unroll
          for (int k = 0; k < 4; ++k) put(piece_v((4 * i + k) ^ (second * 4)), codes_f16(w[k], mm, shift));
        }
        fence_proxy_async_smem();
      }

      // ---- scores ----
      wait_products();
      wait_phase(&keys_bar, step_phase, dead, p);  // (complete: the products were issued after it)
      uint32_t t[T2];
      const int pos0 = step * TOK + half * T2;  // below 2^31 - 1024
      const bool masked = (long long)step * TOK + TOK > see_least;
      float top = -INFINITY;
      auto score = [&](auto with_mask) {
        constexpr bool kMasked = decltype(with_mask)::value;
        float undo = 1.f;
        if constexpr (F32) undo = row_undo[row];
        const Pair undo2 = pair_of(undo, undo);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          uint32_t u[T2];
          tmem_load(t_s + g * TOK, u);
          const float q_sum = row_sum[g * kRows + row];
          const Pair q2 = pair_of(q_sum, q_sum);
#pragma unroll
          for (int j = 0; j < T2; j += 4) {
            Pair a[2], b[2], x[2];
            load_pairs(tok_a + turn + g * TOK + half * T2 + j, a);
            load_pairs(tok_b + turn + g * TOK + half * T2 + j, b);
            if (g == 0) load_pairs(tok_l + turn + half * T2 + j, x);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const int i = j + 2 * k;
              if (g > 0) x[k] = pair_of(__uint_as_float(t[i]), __uint_as_float(t[i + 1]));
              Pair s = pair_of(__uint_as_float(u[i]), __uint_as_float(u[i + 1]));
              if (F32) s = mul2(s, undo2);
              float2 y = values_of(fma2(a[k], s, fma2(b[k], q2, x[k])));
              if (g == NG - 1) {
                if (kMasked && pos0 + i >= see) y.x = -INFINITY;
                if (kMasked && pos0 + i + 1 >= see) y.y = -INFINITY;
                top = fmaxf(top, fmaxf(y.x, y.y));
              }
              t[i] = __float_as_uint(y.x);
              t[i + 1] = __float_as_uint(y.y);
            }
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
#pragma unroll
        for (int g = 0; g < NG; ++g) off[g] *= fall;
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
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          Pair l2 = pair_of(0.f, 0.f), off2 = l2;  // of the step
#pragma unroll
          for (int c = 0; c < T2 / 32; ++c) {
            uint32_t hi[16], lo[16];
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
              Pair inv[2], v[2], d[2];
              if (g == 0) load_pairs(tok_i + turn + half * T2 + c * 32 + j, inv);
              load_pairs(tok_v + turn + g * TOK + half * T2 + c * 32 + j, v);
              if (NG > 1) load_pairs(tok_d + turn + g * TOK + half * T2 + c * 32 + j, d);
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const int i = c * 32 + j + 2 * k;
                Pair x = add2(pair_of(__uint_as_float(t[i]), __uint_as_float(t[i + 1])), r2);
                if (NG > 1) x = add2(x, d[k]);
                float2 w = values_of(x);
                w.x = ex2(w.x);
                w.y = ex2(w.y);
                if (kMasked) {  // what the numbers of hidden tokens are does not matter
                  const bool hide_x = pos0 + i >= see, hide_y = pos0 + i + 1 >= see;
                  const float2 b = values_of(v[k]);
                  v[k] = pair_of(hide_x ? 0.f : b.x, hide_y ? 0.f : b.y);
                  if (g == 0) {
                    const float2 a = values_of(inv[k]);
                    inv[k] = pair_of(hide_x ? 0.f : a.x, hide_y ? 0.f : a.y);
                  }
                }
                const Pair w2 = pair_of(w.x, w.y);
                if (g == 0) l2 = fma2(w2, inv[k], l2);
                off2 = fma2(w2, v[k], off2);
                const uint32_t h = pack_f16(w.x, w.y);
                const float2 rest = values_of(add2(w2, pair_of(-half_lo(h), -half_hi(h))));
                hi[j / 2 + k] = h;
                lo[j / 2 + k] = pack_f16(rest.x, rest.y);
              }
            }
            tmem_store16(t_p + g * TOK + c * 16, hi);
            tmem_store16(t_p + g * TOK + T2 + c * 16, lo);
          }
          const float2 a = values_of(l2), b = values_of(off2);
          if (g == 0) l += a.x + a.y;
          off[g] += b.x + b.y;
        }
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
          constexpr uint32_t idesc = umma_idesc_f16(kRows, G) | 1u << 16;  // B by rows of the k dimension
          const uint64_t b = umma_smem_desc(v_at, 1024, H * 1024, 2);
#pragma unroll
          for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int kk = 0; kk < TOK / 16; ++kk) {
              const uint64_t d = b + (uint64_t)((kk * (H * 2048) + g * (G / 64) * 1024) >> 4);
              const uint32_t o = tmem + kO + g * G, w = tmem + g * TOK + 8 * kk;
              umma_f16_ts(o, w, d, idesc, !fresh || kk > 0);
              umma_f16_ts(o, w + T2, d, idesc, 1);
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
    const float g = aside_ref == ref ? 1.f : ex2(aside_ref - ref);  // (neither has one yet: 1)
    if (aside) l = fmaf(aside_l(), g, l);
    row_max[half * kRows + row] = l;
#pragma unroll
    for (int y = 0; y < NG; ++y) aside_off(y) = aside ? fmaf(aside_off(y), g, off[y]) : off[y];
    __syncthreads();
    l += row_max[(1 - half) * kRows + row];
    const bool whole = cur.c0 == 0 && cur.c1 == cur.steps;
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
      const float* offs = row_off + (half * (D / 2) + c) / G * 2 * kRows + row;
      const float shift = offs[0] + offs[kRows];
      float4 x[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        x[k] = make_float4(__uint_as_float(o[4 * k]) + shift, __uint_as_float(o[4 * k + 1]) + shift,
                           __uint_as_float(o[4 * k + 2]) + shift, __uint_as_float(o[4 * k + 3]) + shift);
        float4* kept = set_aside + (c / 4 + k) * kRows;
        if (aside) add_scaled(x[k], *kept, g);
        if (!whole) *kept = x[k];
      }
      if (whole && row < rows) store_rows<TYPE, 4>(p.o, o_at + c, x, l, over);
    }
    if (!whole && half == 0) {
      float* num = sums + ((size_t)blockIdx.x * 2 + slot) * kSlot + kRows * D + 2 * row;
      num[0] = ref;
      num[1] = l;
    }
    if (!whole && cur.c0 == 0 && tid == 0)
      parts[blockIdx.x] = Part{cur.s.first, rows, cur.head, (int)((at + cur.steps - 1) / r.length - blockIdx.x + 1), row0,
                               slot, 0, 0};
    at += cur.c1 - cur.c0;
    if (at >= r.stop) break;
    next_tile<kRows>(p, per, at, r.stop, cur);
    tcgen05_fence_before();
    __syncthreads();  // the rows' numbers have been read
  }
  // After a wait that gave up products may be under way.  They read this block's shared memory and write its
  // tensor memory, which is another's next: they are waited for, a millisecond at least.
  if (warp == 0 && __any_sync(0xffffffffu, dead)) {
    if (elect_one()) umma_commit(&all_bar);  // of all that this lane has issued
    __syncwarp();
    const uint64_t t0 = global_timer_ns(), most = p.timeout_ns > 1000000ull ? p.timeout_ns : 1000000ull;
    while (!mbar_try_wait(&all_bar, 0) && global_timer_ns() - t0 < most) {
    }
    __syncwarp();
  }
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 0) tmem_dealloc(tmem, M::kTmem);
}

// Joins the parts of the tile that begins in the run of CTA blockIdx.x, kJoinDims dimensions of it: a
// thread a row, four parts under way at a time.
constexpr int kJoinDims = 16, kJoinParts = 4;
template <int D, int TYPE>
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
  store_rows<TYPE, V>(p.o, at, v, sum, over);
}

template <int D, int G, int TYPE>
cudaError_t launch(Kv4AttentionParams p, int sm_count, cudaStream_t st) {
  using M = Form<D, G, TYPE>;
  constexpr int smem = M::kBytes, kMaxDevices = 64;
  static std::atomic<unsigned> asked[kMaxDevices];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const unsigned gen = attr_generation(dev) + 1;
  if (dev >= kMaxDevices || asked[dev].load(std::memory_order_acquire) != gen) {
    e = cudaFuncSetAttribute(kv4_prompt_kernel<D, G, TYPE>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    if (dev < kMaxDevices) asked[dev].store(gen, std::memory_order_release);
  }
  const int ctas = sm_count * M::kCtas;
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
  e = cudaLaunchKernelEx(&cfg, kv4_prompt_kernel<D, G, TYPE>, p);
  if (e != cudaSuccess) return e;
  cfg.dynamicSmemBytes = 0;
  cfg.gridDim = dim3((unsigned)ctas, D / kJoinDims);
  cfg.blockDim = dim3(kRows);
  return cudaLaunchKernelEx(&cfg, kv4_prompt_join_kernel<D, TYPE>, p);
}

template <int D, int G>
cudaError_t launch(const Kv4AttentionParams& p, int dtype, int sm_count, cudaStream_t st) {
  if (dtype == kTypeF32) return launch<D, G, kTypeF32>(p, sm_count, st);
  return dtype == kTypeBF16 ? launch<D, G, kTypeBF16>(p, sm_count, st) : launch<D, G, kTypeF16>(p, sm_count, st);
}

}  // namespace

// On the mean enough rows a sequence.  Against tiles of eight rows, four heads a group of 128, 16 x 2000
// positions with 32 rows take 63 us instead of 52, with 48 64 instead of 73, with 128 69 instead of 168
// (f32: 86 and 52, 64 rows 90 and 91, 98 and 168; 256 dimensions in two groups: 142 and 105, 143 and 148;
// of f32 with 64 rows 196 and 194); 60000 positions 108 and 76, 108 and 106, 112 and 257.  A step is long, so little
// work in all wants more rows: one sequence of 3000, by the table's reach, with 128 rows 33 us instead of 27, with
// 256 33 instead of 40 (f32: 41 and 27, 43 and 40; 256 dimensions: 35 and 45 with 128, 34 and 29 with 64; f32 of them
// 45 and 45 with 128).
bool kv4_prompt_takes(const Kv4AttentionParams& p, int dtype) {
  const bool wide = dtype == kTypeF32, large = p.cache.head_dim == 256;
  const long long rows = (long long)p.tokens * (p.q_heads / p.cache.kv_heads);
  const long long tiles = (rows / kRows + p.batch) * p.cache.kv_heads;
  const long long steps = (((long long)p.max_blocks << p.cache.shift) + kStep - 1) / kStep + kTileCost;
  const long long few = (wide ? 288 : 160) / (large ? 2 : 1), many = wide ? 64 : 48;
  return rows >= few * p.batch || (rows >= many * p.batch && tiles * steps >= 600);
}

size_t kv4_prompt_workspace(int head_dim, int sm_count) {
  return attention_workspace(sm_count * (head_dim == 256 ? 1 : 2), kRows, head_dim);
}

cudaError_t launch_kv4_prompt(Kv4AttentionParams p, int dtype, int sm_count, cudaStream_t st) {
  const int d = p.cache.head_dim, g = p.cache.group;
  if (d == 64) return launch<64, 64>(p, dtype, sm_count, st);
  if (d == 128) return g == 64 ? launch<128, 64>(p, dtype, sm_count, st) : launch<128, 128>(p, dtype, sm_count, st);
  return g == 64 ? launch<256, 64>(p, dtype, sm_count, st) : launch<256, 128>(p, dtype, sm_count, st);
}

}  // namespace tk
