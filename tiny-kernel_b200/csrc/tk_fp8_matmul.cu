// tk_fp8_matmul.cu -- rows of e4m3 codes times a weight of e4m3 codes, a scale for each block of 128 of k:
//
//   out[m][n] = sum over blocks b of  a_scales[m][b] w_scales[n / 128][b]  sum of a[m][k] w[n][k] in b
//
// The inner sums are products of 8-bit numbers on tcgen05, a block of k at a time into an accumulator of its own
// in tensor memory; the outer sum, with the scales, is f32 in registers.
#include <algorithm>
#include <atomic>

#include "tk_elements.cuh"
#include "tk_fp8.h"
#include "tk_internal.h"
#include "tk_kv4.h"
#include "tk_ptx.cuh"

namespace tk {
namespace {

constexpr unsigned kErrFp8Wait = 128u;  // a copy or a product never completed

// Waits, all lanes of a warp, for the phase of `bar`; gives up, for good, after timeout_ns.  The timer is read once in many
// tries, since a read takes longer than a phase should be noticed late.  A lane may give up where another, that read the timer
// earlier or later, sees the phase complete: what they do next goes by agreed().
__device__ __forceinline__ void wait_phase(uint64_t* bar, uint32_t phase, bool& dead, const Fp8MatmulParams& p) {
  if (dead || mbar_try_wait(bar, phase)) return;
  uint64_t t0 = 0;
  bool late = false;
  for (uint32_t tries = 1; !mbar_try_wait(bar, phase); ++tries) {
    if (late) {
      atomicOr(p.err, kErrFp8Wait);
      dead = true;
      return;
    }
    if (tries % 64 != 0) continue;
    const uint64_t now = global_timer_ns();
    if (t0 == 0) t0 = now;
    late = now - t0 > p.timeout_ns;
  }
}
// Whether a lane of the warp gave up: then all do, since instructions of whole warps follow.
__device__ __forceinline__ bool agreed(bool dead) { return __any_sync(0xffffffffu, dead); }

// D[tmem] (+)= A[smem] x B[smem], e4m3, f32 sums, 32 of k.  The instruction's word is that of f16: type 0 is e4m3 here.
__device__ __forceinline__ void umma_e4m3(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, {%5, %6, %7, %8}, p;\n\t}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(0), "r"(0), "r"(0), "r"(0));
}

#define TK_R4(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3])
// 16 consecutive columns of the warp's 32 lanes; complete after tmem_ld_wait.
__device__ __forceinline__ void tmem_ld16(uint32_t at, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15}, [%16];"
      : TK_R4(r, 0), TK_R4(r, 4), TK_R4(r, 8), TK_R4(r, 12)
      : "r"(at));
}
#undef TK_R4

__device__ __forceinline__ void store_out(const Fp8MatmulParams& p, long long at, float v) {
  if (p.dtype == kTypeF32)
    static_cast<float*>(p.out)[at] = v;
  else if (p.dtype == kTypeBF16)
    static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(v);
  else
    static_cast<__half*>(p.out)[at] = __float2half_rn(v);
}

// n of four values of a row, on the boundary of four of them or not.
template <class T>
__device__ __forceinline__ void store_four(T* dst, int n, const float4& v) {
  const float e[4] = {v.x, v.y, v.z, v.w};
  if (n >= 4 && reinterpret_cast<uintptr_t>(dst) % (4 * sizeof(T)) == 0) {
    struct alignas(4 * sizeof(T)) Four {
      T e[4];
    } y;
#pragma unroll
    for (int i = 0; i < 4; ++i) y.e[i] = from_f32<T>(e[i]);
    *reinterpret_cast<Four*>(dst) = y;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) dst[i] = from_f32<T>(e[i]);
  }
}
__device__ __forceinline__ void store_four(const Fp8MatmulParams& p, long long at, int n, const float4& v) {
  if (p.dtype == kTypeF32)
    store_four(static_cast<float*>(p.out) + at, n, v);
  else if (p.dtype == kTypeBF16)
    store_four(static_cast<__nv_bfloat16*>(p.out) + at, n, v);
  else
    store_four(static_cast<__half*>(p.out) + at, n, v);
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Four values of a CTA of the cluster.  (Not ordered by the compiler among others: several travel at once; the barrier
// before them and the one after are.)
__device__ __forceinline__ float4 ld_peer(uint32_t addr, uint32_t rank) {
  uint32_t at;
  float4 v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at));
  return v;
}

// ---- few rows ------------------------------------------------------------------------------------------
//
// The weight's rows are the product's 128 rows, the activations, NT at the most, its columns: the weight is read once, by
// as many CTAs as keep memory busy, two a SM.  Where there are fewer tiles than that, the CTAs of a cluster share a tile's
// blocks of k and add their sums through shared memory, in the order of their ranks; where there are more, a CTA walks over
// its tiles and its copies go on through their ends.  Bound by memory, and below some 60 MB by the way to the first
// product and from the last: 48 x 4096 x 128256 (525 MB of weight) 92 to 110 us, 4.8 to 5.7 TB/s; 1 x 4096 x 14336 (59 MB)
// 12.6, 4.7 TB/s, with a CTA on 112 of 148 SMs; 32 x 14336 x 4096 14.0, 256 CTAs on 148 SMs.
//
// Waits of a cluster's CTAs for one another need all of them to get their tensor memory.  They do: two CTAs of this form
// have the 512 columns of a SM at most and leave no shared memory for a third, those below fill a SM's shared memory
// alone, and no other kernel of the framework that has tensor memory waits for another CTA while it holds it.

constexpr int kMaxSplit = 8;

template <int NT>
struct Few {
  static constexpr int kStep = NT <= 32 ? 2 : 1;       // blocks of k between two waits
  static constexpr int kGroups = NT >= 64 ? 2 : 1;     // warpgroups of sums, half of the columns each
  static constexpr int kCols = NT / kGroups, kChunk = kCols < 32 ? kCols : 32;
  static constexpr int kCtas = 2;                      // of an SM
  static constexpr int kThreads = 64 + 128 * kGroups;  // a warp of copies, one of products, those of sums
  static constexpr int kSums = 4;                      // steps in tensor memory
  static constexpr uint32_t kColumns = kSums * kStep * NT;
  static constexpr int kBlockBytes = (128 + NT) * kFp8Block, kStageBytes = kStep * kBlockBytes;
  // Half of a SM's shared memory, also where there is a CTA for each only: the next launch's are set up beside them
  // (with all of it, 1 x 4096 x 14336 and 16 x 4096 x 4096 12.8 and 6.3 us instead of 12.4 and 6.0).
  static constexpr int kStages = 110 * 1024 / kStageBytes, kBytes = kStages * kStageBytes + 1024;
  static_assert(NT * 512 <= kStages * kStageBytes, "shared memory");
};

template <int NT>
__global__ void __launch_bounds__(Few<NT>::kThreads, Few<NT>::kCtas) fp8_few_kernel(const __grid_constant__ CUtensorMap a_map,
                                                                       const __grid_constant__ CUtensorMap w_map,
                                                                       Fp8MatmulParams p, int split, int tiles) {
  using M = Few<NT>;
  constexpr int KS = M::kStep, NC = M::kCols, CH = M::kChunk;
  extern __shared__ uint8_t dynamic[];
  __shared__ uint64_t full[M::kStages], empty[M::kStages], sums_full[M::kSums], sums_empty[M::kSums], drained;
  __shared__ uint32_t tmem_slot;
  __shared__ __align__(16) float factors[4 * M::kGroups][2][KS][NC];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* smem = dynamic + ((1024u - (smem_addr(dynamic) & 1023u)) & 1023u);
  const int rank = blockIdx.x % split, first = blockIdx.x / split, stride = gridDim.x / split;  // of tiles
  const int blocks = (p.k + kFp8Block - 1) / kFp8Block;
  const int b0 = (int)((long long)blocks * rank / split), b1 = (int)((long long)blocks * (rank + 1) / split);
  if (threadIdx.x == 0) {
    for (int s = 0; s < M::kStages; ++s) mbar_init(&full[s], 1), mbar_init(&empty[s], 1);
    for (int s = 0; s < M::kSums; ++s) mbar_init(&sums_full[s], 1), mbar_init(&sums_empty[s], 4 * M::kGroups);
    mbar_init(&drained, 1);
    fence_mbar_init();
  }
  after_previous();
  if (warp == 1) tmem_alloc(&tmem_slot, M::kColumns);
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = tmem_slot;
  bool dead = false;
  int issued = 0;
  unsigned long long acc[NC / 2];
  const int quarter = warp & 3, group = (warp - 2) >> 2, row = quarter * 32 + lane;
  if (warp == 0) {
    const uint64_t once = l2_evict_first(), often = l2_evict_last();
    int stage = 0;
    uint32_t phase = 1;  // a barrier's phase before its first counts as complete
    for (int t = first; t < tiles && !dead; t += stride) {
      for (int b = b0; b < b1; b += KS) {
        wait_phase(&empty[stage], phase, dead, p);
        dead = agreed(dead);
        if (dead) break;
        const int n = min(KS, b1 - b);
        if (elect_one()) {
          uint8_t* to = smem + stage * M::kStageBytes;
          mbar_arrive_expect_tx(&full[stage], n * M::kBlockBytes);
          for (int i = 0; i < n; ++i) {
            tma_load_2d(to + i * 16384, &w_map, &full[stage], (b + i) * kFp8Block, t * 128, once);
            tma_load_2d(to + KS * 16384 + i * NT * kFp8Block, &a_map, &full[stage], (b + i) * kFp8Block, 0, often);
          }
        }
        __syncwarp();
        ++issued;
        if (++stage == M::kStages) stage = 0, phase ^= 1;
      }
    }
  } else if (warp == 1) {
    constexpr uint32_t idesc = umma_idesc_f16(128, NT);
    const uint64_t w0 = umma_smem_desc(smem_addr(smem), 16, 1024, 2);
    const uint64_t a0 = umma_smem_desc(smem_addr(smem) + KS * 16384, 16, 1024, 2);
    int stage = 0, d = 0;
    uint32_t phase = 0, sums_phase = 1;
    for (int t = first; t < tiles && !dead; t += stride)
      for (int b = b0; b < b1; b += KS) {
        const int n = min(KS, b1 - b);
        wait_phase(&full[stage], phase, dead, p);
        wait_phase(&sums_empty[d], sums_phase, dead, p);
        dead = agreed(dead);
        if (dead) break;
        tcgen05_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int i = 0; i < KS; ++i) {
            if (i >= n) break;
            const uint64_t w = w0 + ((stage * M::kStageBytes + i * 16384) >> 4);
            const uint64_t a = a0 + ((stage * M::kStageBytes + i * NT * kFp8Block) >> 4);
#pragma unroll
            for (int k = 0; k < 4; ++k) umma_e4m3(tmem + (d * KS + i) * NT, w + 2 * k, a + 2 * k, idesc, k > 0);
          }
          umma_commit(&sums_full[d]);
          umma_commit(&empty[stage]);
        }
        __syncwarp();
        if (++stage == M::kStages) stage = 0, phase ^= 1;
        if (++d == M::kSums) d = 0, sums_phase ^= 1;
      }
  } else {
    const uint32_t from = tmem + ((uint32_t)(quarter * 32) << 16) + group * NC;
    float(&mine)[2][KS][NC] = factors[warp - 2];
    constexpr int kEach = (NC + 31) / 32;
    int d = 0, turn = 0;
    uint32_t phase = 0;
    for (int t = first; t < tiles && !dead; t += stride) {
      const float* w_scale = p.w_scales + (long long)t * blocks;
#pragma unroll
      for (int j = 0; j < NC / 2; ++j) acc[j] = 0;
      float next[KS][kEach], next_w[KS];  // multiplied when they are needed: not waited for before that
      auto fetch = [&](int b) {
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          next_w[i] = b + i < b1 ? w_scale[b + i] : 0.f;
#pragma unroll
          for (int e = 0; e < kEach; ++e) {
            const int j = e * 32 + lane, token = group * NC + j;
            next[i][e] = b + i < b1 && j < NC && token < p.m ? p.a_scales[(long long)token * blocks + b + i] : 0.f;
          }
        }
      };
      fetch(b0);
      for (int b = b0; b < b1; b += KS) {
        float(&now)[KS][NC] = mine[turn];
        turn ^= 1;
#pragma unroll
        for (int i = 0; i < KS; ++i)
#pragma unroll
          for (int e = 0; e < kEach; ++e)
            if (e * 32 + lane < NC) now[i][e * 32 + lane] = next[i][e] * next_w[i];
        if (b + KS < b1) fetch(b + KS);
        const int n = min(KS, b1 - b);
        wait_phase(&sums_full[d], phase, dead, p);
        __syncwarp();  // (the factors, too)
        dead = agreed(dead);
        if (dead) break;
        tcgen05_fence_after();
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          if (i >= n) break;
#pragma unroll
          for (int c = 0; c < NC; c += CH) {
            uint32_t v[CH];
#pragma unroll
            for (int x = 0; x < CH; x += 16) tmem_ld16(from + (d * KS + i) * NT + c + x, v + x);
            tmem_ld_wait();
            if (c + CH == NC && i + 1 == n) {  // all read: the accumulators are free
              tcgen05_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&sums_empty[d]);
            }
            const float4* f = reinterpret_cast<const float4*>(&now[i][c]);
#pragma unroll
            for (int j = 0; j < CH / 4; ++j) {
              const float4 g = f[j];
              unsigned long long* to = &acc[c / 2 + 2 * j];
              to[0] = fma2(pair_of(__uint_as_float(v[4 * j]), __uint_as_float(v[4 * j + 1])), pair_of(g.x, g.y), to[0]);
              to[1] = fma2(pair_of(__uint_as_float(v[4 * j + 2]), __uint_as_float(v[4 * j + 3])), pair_of(g.z, g.w), to[1]);
            }
          }
        }
        if (++d == M::kSums) d = 0, phase ^= 1;
      }
      if (split > 1 || dead) break;  // one tile a cluster
      const int n = t * 128 + row;
      if (n < p.n) {
#pragma unroll
        for (int j = 0; j < NC / 2; ++j) {
          const float2 v = values_of(acc[j]);
          const int token = group * NC + 2 * j;
          if (token < p.m) store_out(p, token * p.out_stride + n, v.x);
          if (token + 1 < p.m) store_out(p, (token + 1) * p.out_stride + n, v.y);
        }
      }
    }
  }
  // After a wait that gave up: what is in flight completes before its memory is given back.
  if (__syncthreads_or(dead)) {
    bool late = false;
    if (warp == 0)
      for (int s = max(0, issued - M::kStages); s < issued; ++s)
        wait_phase(&full[s % M::kStages], (s / M::kStages) & 1, late, p);
    if (warp == 1) {
      if (elect_one()) umma_commit(&drained);
      __syncwarp();
      wait_phase(&drained, 0, late, p);
    }
    __syncwarp();
    dead = true;
    __syncthreads();
  }
  if (split > 1) {
    float* sums = reinterpret_cast<float*>(smem);  // [NT][128]
    if (warp >= 2) {
#pragma unroll
      for (int j = 0; j < NC / 2; ++j) {
        const float2 v = values_of(acc[j]);
        sums[(group * NC + 2 * j) * 128 + row] = v.x;
        sums[(group * NC + 2 * j + 1) * 128 + row] = v.y;
      }
    }
    cluster_sync();
    // the tokens' columns over the CTAs, four rows a thread, all CTAs' values at once
    const int j0 = p.m * rank / split, j1 = p.m * (rank + 1) / split;
    for (int i = threadIdx.x; !dead && i < (j1 - j0) * 32; i += M::kThreads) {
      const int j = j0 + i / 32, row4 = i % 32 * 4, n = first * 128 + row4;
      if (n >= p.n) continue;
      const uint32_t from = smem_addr(sums + j * 128 + row4);
      float4 v[kMaxSplit];
#pragma unroll
      for (int r = 0; r < kMaxSplit; ++r)
        if (r < split) v[r] = ld_peer(from, r);
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int r = 0; r < kMaxSplit; ++r)
        if (r < split) sum.x += v[r].x, sum.y += v[r].y, sum.z += v[r].z, sum.w += v[r].w;
      store_four(p, j * p.out_stride + n, p.n - n, sum);
    }
    __syncwarp();
    cluster_sync();
  }
  if (warp == 1) {
    tcgen05_fence_after();
    tmem_dealloc(tmem, M::kColumns);
  }
}

template <int NT>
cudaError_t launch_few(const Fp8MatmulParams& p, const Fp8MatmulPlan& plan, const CUtensorMap& a_map,
                       const CUtensorMap& w_map, int sm_count, cudaStream_t st) {
  using M = Few<NT>;
  constexpr int kMaxDevices = 64;
  static std::atomic<unsigned> asked[kMaxDevices];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const unsigned gen = attr_generation(dev) + 1;
  if (dev >= kMaxDevices || asked[dev].load(std::memory_order_acquire) != gen) {
    e = cudaFuncSetAttribute(fp8_few_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, M::kBytes);
    if (e != cudaSuccess) return e;
    if (dev < kMaxDevices) asked[dev].store(gen, std::memory_order_release);
  }
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)plan.split;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)fp8_matmul_places(plan, p.m, p.n, sm_count));
  cfg.blockDim = dim3(M::kThreads);
  cfg.dynamicSmemBytes = M::kBytes;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = plan.split > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, fp8_few_kernel<NT>, a_map, w_map, p, plan.split, (p.n + 127) / 128);
}

// ---- tiles with the activations as rows ------------------------------------------------------------------

constexpr int kTileGroup = 8;  // tiles of rows that share the weight's tiles at a time, for L2
constexpr int kPatch = 32 * 33 * 4;  // bytes of a warp's corner of shared memory, for rows off their 32-byte boundary

struct Tile {
  int m, n;
};
__device__ __forceinline__ Tile tile_of(int t, int tiles_m, int tiles_n) {
  const int group = t / (kTileGroup * tiles_n), first = group * kTileGroup, rows = min(kTileGroup, tiles_m - first);
  const int r = t - group * kTileGroup * tiles_n;
  return {first + r % rows, r / rows};
}

// 32 values of a row.
template <class T>
__device__ __forceinline__ void store_32(T* dst, const float (&v)[32]) {
  constexpr int kWords = 32 * sizeof(T) / 32;
#pragma unroll
  for (int w = 0; w < kWords; ++w) {
    uint32_t y[8];
    T* e = reinterpret_cast<T*>(y);
#pragma unroll
    for (int j = 0; j < 32 / (int)sizeof(T); ++j) e[j] = from_f32<T>(v[w * (32 / sizeof(T)) + j]);
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(dst + w * (32 / sizeof(T))), "r"(y[0]), "r"(y[1]),
                 "r"(y[2]), "r"(y[3]), "r"(y[4]), "r"(y[5]), "r"(y[6]), "r"(y[7])
                 : "memory");
  }
}
// 32 consecutive values of a row a lane, from column `at` on: whole sectors, or through the warp's corner of shared
// memory where rows are off their boundary.
template <class T>
__device__ __forceinline__ void store_rows(const Fp8MatmulParams& p, int row, int at, bool wide, float* patch,
                                           const float (&v)[32]) {
  const int lane = threadIdx.x & 31;
  if (wide && at + 32 <= p.n) {
    if (row < p.m) store_32(static_cast<T*>(p.out) + row * p.out_stride + at, v);
    return;
  }
#pragma unroll
  for (int j = 0; j < 32; ++j) patch[lane * 33 + j] = v[j];
  __syncwarp();
  const int rows = min(32, p.m - (row - lane));
  T* corner = static_cast<T*>(p.out) + (long long)(row - lane) * p.out_stride + at + lane;
  if (at + lane < p.n)
    for (int r = 0; r < rows; ++r) corner[r * p.out_stride] = from_f32<T>(patch[r * 33 + lane]);
  __syncwarp();
}

// ---- some rows -----------------------------------------------------------------------------------------
//
// Tiles of 128 rows by 128 or 256 of the weight's: a thread adds half of a row, whose scale is one number a block (in the
// form for few rows it is one for each column, read from shared memory for each product).  Accumulators fill tensor
// memory.  CTAs of a cluster share a tile's k (of 128 columns), or walk over tiles, as above.  Bound by the chain of one
// block after the other (0.4 to 0.5 us: products, word, sums, word back) where a CTA has a tile or two: 777 x 2000 x 5003
// 17.2 us over the same buffers, of which tiles take 8, and 21.6 with operands and outputs in memory.

// The registers of a launch of three warpgroups, 168 for each thread, are handed from the first group, of copies and
// products, to the two of sums, where a thread holds 128 of them: 40 and 2 x 232 of 3 x 168.
constexpr int kEvenRegs = 168, kFewRegs = 40, kMoreRegs = 232;
static_assert(kFewRegs + 2 * kMoreRegs <= 3 * kEvenRegs, "the groups' shares");

template <int COLS>
struct Some {
  static constexpr int kFirst = COLS == 256 ? 4 : 2;     // warps before those of sums: of copies, of products
  static constexpr int kThreads = kFirst * 32 + 256, kHalf = COLS / 2, kSums = 512 / COLS;
  static constexpr int kStageBytes = (128 + COLS) * kFp8Block, kStages = 192 * 1024 / kStageBytes;
  static constexpr int kBytes = kStages * kStageBytes + 8 * kPatch + 1024;
};
constexpr int kSomePitch = 132;  // floats of a row of the exchange
static_assert(128 * kSomePitch * 4 <= Some<128>::kStages * Some<128>::kStageBytes, "shared memory");

template <class T, int COLS>
__global__ void __launch_bounds__(Some<COLS>::kThreads, 1) fp8_some_kernel(const __grid_constant__ CUtensorMap a_map,
                                                                           const __grid_constant__ CUtensorMap w_map,
                                                                           Fp8MatmulParams p, int split, int tiles_m,
                                                                           int tiles_n, int wide) {
  using M = Some<COLS>;
  extern __shared__ uint8_t dynamic[];
  __shared__ uint64_t full[M::kStages], empty[M::kStages], sums_full[M::kSums], sums_empty[M::kSums], drained;
  __shared__ uint32_t tmem_slot;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* smem = dynamic + ((1024u - (smem_addr(dynamic) & 1023u)) & 1023u);
  const int rank = blockIdx.x % split, first = blockIdx.x / split, stride = gridDim.x / split, tiles = tiles_m * tiles_n;
  const int blocks = (p.k + kFp8Block - 1) / kFp8Block;
  const int b0 = (int)((long long)blocks * rank / split), b1 = (int)((long long)blocks * (rank + 1) / split);
  if (threadIdx.x == 0) {
    for (int s = 0; s < M::kStages; ++s) mbar_init(&full[s], 1), mbar_init(&empty[s], 1);
    for (int s = 0; s < M::kSums; ++s) mbar_init(&sums_full[s], 1), mbar_init(&sums_empty[s], 8);
    mbar_init(&drained, 1);
    fence_mbar_init();
  }
  after_previous();
  if (warp == 1) tmem_alloc(&tmem_slot, 512);
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = tmem_slot;
  bool dead = false;
  int issued = 0;
  unsigned long long acc[M::kHalf / 2];
  const int quarter = warp & 3, half = (warp - M::kFirst) >> 2;
  if (COLS == 256 && warp < M::kFirst) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewRegs));
  if (warp == 0) {
    const uint64_t once = tiles_m == 1 ? l2_evict_first() : l2_evict_last(), often = l2_evict_last();
    int stage = 0;
    uint32_t phase = 1;  // a barrier's phase before its first counts as complete
    for (int t = first; t < tiles && !dead; t += stride) {
      const Tile tile = tile_of(t, tiles_m, tiles_n);
      for (int b = b0; b < b1; ++b) {
        wait_phase(&empty[stage], phase, dead, p);
        dead = agreed(dead);
        if (dead) break;
        if (elect_one()) {
          uint8_t* to = smem + stage * M::kStageBytes;
          mbar_arrive_expect_tx(&full[stage], M::kStageBytes);
          tma_load_2d(to, &a_map, &full[stage], b * kFp8Block, tile.m * 128, often);
          tma_load_2d(to + 128 * kFp8Block, &w_map, &full[stage], b * kFp8Block, tile.n * COLS, once);
        }
        __syncwarp();
        ++issued;
        if (++stage == M::kStages) stage = 0, phase ^= 1;
      }
    }
  } else if (warp == 1) {
    constexpr uint32_t idesc = umma_idesc_f16(128, COLS);
    const uint64_t a0 = umma_smem_desc(smem_addr(smem), 16, 1024, 2);
    const uint64_t w0 = umma_smem_desc(smem_addr(smem) + 128 * kFp8Block, 16, 1024, 2);
    int stage = 0, d = 0;
    uint32_t phase = 0, sums_phase = 1;
    for (int t = first; t < tiles && !dead; t += stride)
      for (int b = b0; b < b1; ++b) {
        const uint64_t a = a0 + stage * (M::kStageBytes >> 4), w = w0 + stage * (M::kStageBytes >> 4);
        const uint32_t to = tmem + d * COLS;
        wait_phase(&full[stage], phase, dead, p);
        wait_phase(&sums_empty[d], sums_phase, dead, p);
        dead = agreed(dead);
        if (dead) break;
        tcgen05_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < 4; ++k) umma_e4m3(to, a + 2 * k, w + 2 * k, idesc, k > 0);
          umma_commit(&sums_full[d]);
          umma_commit(&empty[stage]);
        }
        __syncwarp();
        if (++stage == M::kStages) stage = 0, phase ^= 1;
        if (++d == M::kSums) d = 0, sums_phase ^= 1;
      }
  } else if (warp >= M::kFirst) {
    if (COLS == 256) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kMoreRegs));
    const uint32_t from = tmem + ((uint32_t)(quarter * 32) << 16) + half * M::kHalf;
    float* patch = reinterpret_cast<float*>(smem + M::kStages * M::kStageBytes + (warp - M::kFirst) * kPatch);
    int d = 0;
    uint32_t phase = 0;
    for (int t = first; t < tiles && !dead; t += stride) {
      const Tile tile = tile_of(t, tiles_m, tiles_n);
      const int row = tile.m * 128 + quarter * 32 + lane, col = tile.n * COLS + half * M::kHalf;
      const float* a_scale = p.a_scales + (long long)min(row, p.m - 1) * blocks;
      const float* w_scale = p.w_scales + (long long)min(col / kFp8Block, (p.n - 1) / kFp8Block) * blocks;
#pragma unroll
      for (int j = 0; j < M::kHalf / 2; ++j) acc[j] = 0;
      // (multiplied when they are needed: not waited for before that)
      float next_a = a_scale[b0], next_w = w_scale[b0];
      for (int b = b0; b < b1; ++b) {
        const float scale = next_a * next_w;
        const unsigned long long f = pair_of(scale, scale);
        if (b + 1 < b1) next_a = a_scale[b + 1], next_w = w_scale[b + 1];
        const uint32_t at = from + d * COLS;
        wait_phase(&sums_full[d], phase, dead, p);
        dead = agreed(dead);
        if (dead) break;
        tcgen05_fence_after();
#pragma unroll
        for (int c = 0; c < M::kHalf; c += 64) {
          uint32_t v[64];
#pragma unroll
          for (int x = 0; x < 64; x += 16) tmem_ld16(at + c + x, v + x);
          tmem_ld_wait();
          if (c + 64 == M::kHalf) {  // all read: the accumulator is free, whatever is still to be added
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sums_empty[d]);
          }
#pragma unroll
          for (int j = 0; j < 32; ++j)
            acc[c / 2 + j] = fma2(pair_of(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1])), f, acc[c / 2 + j]);
        }
        if (++d == M::kSums) d = 0, phase ^= 1;
      }
      if (split > 1 || dead) break;  // one tile a cluster
#pragma unroll
      for (int c = 0; c < M::kHalf; c += 32) {
        float v[32];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float2 y = values_of(acc[c / 2 + j]);
          v[2 * j] = y.x, v[2 * j + 1] = y.y;
        }
        store_rows<T>(p, row, col + c, wide, patch, v);
      }
    }
  }
  // After a wait that gave up: what is in flight completes before its memory is given back.
  if (__syncthreads_or(dead)) {
    bool late = false;
    if (warp == 0)
      for (int s = max(0, issued - M::kStages); s < issued; ++s)
        wait_phase(&full[s % M::kStages], (s / M::kStages) & 1, late, p);
    if (warp == 1) {
      if (elect_one()) umma_commit(&drained);
      __syncwarp();
      wait_phase(&drained, 0, late, p);
    }
    __syncwarp();
    dead = true;
    __syncthreads();
  }
  if (COLS == 128 && split > 1) {
    const Tile tile = tile_of(first, tiles_m, tiles_n);
    float* sums = reinterpret_cast<float*>(smem);  // [128][pitch]
    if (warp >= M::kFirst) {
      float* mine = sums + (quarter * 32 + lane) * kSomePitch + half * 64;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float2 x = values_of(acc[2 * j]), y = values_of(acc[2 * j + 1]);
        reinterpret_cast<float4*>(mine)[j] = make_float4(x.x, x.y, y.x, y.y);
      }
    }
    cluster_sync();
    // the rows over the CTAs, four columns a thread, all CTAs' values at once
    const int rows = min(128, p.m - tile.m * 128), r0 = rows * rank / split, r1 = rows * (rank + 1) / split;
    for (int i = threadIdx.x; !dead && i < (r1 - r0) * 32; i += M::kThreads) {
      const int r = r0 + i / 32, n = tile.n * 128 + i % 32 * 4;
      if (n >= p.n) continue;
      const uint32_t from = smem_addr(sums + r * kSomePitch + i % 32 * 4);
      float4 v[kMaxSplit];
#pragma unroll
      for (int q = 0; q < kMaxSplit; ++q)
        if (q < split) v[q] = ld_peer(from, q);
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int q = 0; q < kMaxSplit; ++q)
        if (q < split) sum.x += v[q].x, sum.y += v[q].y, sum.z += v[q].z, sum.w += v[q].w;
      store_four(static_cast<T*>(p.out) + (tile.m * 128 + r) * p.out_stride + n, p.n - n, sum);
    }
    __syncwarp();
    cluster_sync();
  }
  if (warp == 1) {
    tcgen05_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// A launch whose groups share out other registers than the kernel has would wait for them for good.
template <class K>
cudaError_t has_even_regs(K kernel) {
  cudaFuncAttributes has{};
  const cudaError_t e = cudaFuncGetAttributes(&has, kernel);
  return e != cudaSuccess ? e : has.numRegs < kEvenRegs ? cudaErrorInvalidKernelImage : cudaSuccess;
}

template <class T, int COLS>
cudaError_t launch_some(const Fp8MatmulParams& p, const Fp8MatmulPlan& plan, const CUtensorMap& a_map,
                        const CUtensorMap& w_map, int sm_count, cudaStream_t st) {
  using M = Some<COLS>;
  constexpr int kMaxDevices = 64;
  static std::atomic<unsigned> asked[kMaxDevices];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const unsigned gen = attr_generation(dev) + 1;
  if (dev >= kMaxDevices || asked[dev].load(std::memory_order_acquire) != gen) {
    if (COLS == 256 && (e = has_even_regs(fp8_some_kernel<T, COLS>)) != cudaSuccess) return e;
    e = cudaFuncSetAttribute(fp8_some_kernel<T, COLS>, cudaFuncAttributeMaxDynamicSharedMemorySize, M::kBytes);
    if (e != cudaSuccess) return e;
    if (dev < kMaxDevices) asked[dev].store(gen, std::memory_order_release);
  }
  const int tiles_m = (p.m + 127) / 128, tiles_n = (p.n + COLS - 1) / COLS;
  const int wide = (reinterpret_cast<uintptr_t>(p.out) | (uintptr_t)(p.out_stride * (long long)sizeof(T))) % 32 == 0;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)plan.split;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)fp8_matmul_places(plan, p.m, p.n, sm_count));
  cfg.blockDim = dim3(M::kThreads);
  cfg.dynamicSmemBytes = M::kBytes;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = plan.split > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, fp8_some_kernel<T, COLS>, a_map, w_map, p, plan.split, tiles_m, tiles_n, wide);
}

// ---- many rows -----------------------------------------------------------------------------------------
//
// The activations are the product's rows, 256 rows of the weight its columns.  Two CTAs share a product of 256 x 256:
// each brings its 128 rows and half of the columns' weight, and has its rows' sums in its tensor memory.  (Alone, a
// CTA would bring 48 KB a block to its 128 x 256 products, and writing and reading them would take shared memory
// longer than the products take.)  A thread adds half of a row in registers, so that its scale is one number a block:
// sum += scale * product.  Two accumulators of 256 columns fill tensor memory: one is added up while the other's
// products run.  Pairs of CTAs walk over the tiles.  8192 x 4096 x 14336: 425 to 450 us in bursts (2.2 PFLOP/s), 480 to
// 520 in long runs, where power limits the clock; the tensor pipe is busy 55 % of the time, and waits for the sums of
// the block before the last (a block's 128 x 256 values through registers take about as long as its products).

constexpr int kManyThreads = 384;  // a warpgroup with a warp of copies and two of products, two warpgroups of sums
constexpr int kManyRows = 256, kManyCols = 256, kManyStages = 6, kManyStageBytes = 2 * 128 * kFp8Block;  // a CTA's part

// The products of a pair, issued by its first CTA.
__device__ __forceinline__ void umma_e4m3_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                               uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate));
}
// Arrives on that barrier of both CTAs when every product issued so far by this thread completes.
__device__ __forceinline__ void umma_commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_addr(bar)),
      "h"((uint16_t)3)
      : "memory");
}
__device__ __forceinline__ void tmem_alloc_pair(uint32_t* slot, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(slot)), "r"(ncols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
__device__ __forceinline__ uint32_t of_first(const void* mine) {  // shared memory of the pair's first CTA
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(at) : "r"(smem_addr(mine)));
  return at;
}
// A box into this CTA's shared memory, counted by a barrier of the first one's.
__device__ __forceinline__ void tma_load_pair(void* dst, const CUtensorMap* map, uint32_t bar, int x, int y,
                                              uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      ".L2::cache_hint [%0], [%1, {%2, %3}], [%4], %5;" ::"r"(smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar), "l"(policy)
      : "memory");
}
__device__ __forceinline__ void arrive_at(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

template <class T>
__global__ void __launch_bounds__(kManyThreads, 1) fp8_many_kernel(const __grid_constant__ CUtensorMap a_map,
                                                                   const __grid_constant__ CUtensorMap w_map,
                                                                   Fp8MatmulParams p, int tiles_m, int tiles_n, int wide) {
  extern __shared__ uint8_t dynamic[];
  __shared__ uint64_t full[kManyStages], empty[kManyStages], sums_full[2], sums_empty[2], drained;
  __shared__ uint32_t tmem_slot;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x & 1, pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  uint8_t* smem = dynamic + ((1024u - (smem_addr(dynamic) & 1023u)) & 1023u);
  const int blocks = (p.k + kFp8Block - 1) / kFp8Block, tiles = tiles_m * tiles_n;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kManyStages; ++s) mbar_init(&full[s], 1), mbar_init(&empty[s], 1);
    for (int s = 0; s < 2; ++s) mbar_init(&sums_full[s], 1), mbar_init(&sums_empty[s], 16);
    mbar_init(&drained, 2);
    fence_mbar_init();
  }
  after_previous();
  if (warp == 1) tmem_alloc_pair(&tmem_slot, 2 * kManyCols);
  tcgen05_fence_before();
  __syncthreads();
  cluster_sync();
  tcgen05_fence_after();
  const uint32_t tmem = tmem_slot;
  bool dead = false;
  int issued = 0;
  if (warp < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewRegs));
  if (warp == 0) {
    const uint64_t often = l2_evict_last();
    int stage = 0;
    uint32_t phase = 1;  // a barrier's phase before its first counts as complete
    for (int t = pair; t < tiles && !dead; t += pairs) {
      const Tile tile = tile_of(t, tiles_m, tiles_n);
      for (int b = 0; b < blocks; ++b) {
        wait_phase(&empty[stage], phase, dead, p);
        dead = agreed(dead);
        if (dead) break;
        if (elect_one()) {
          uint8_t* to = smem + stage * kManyStageBytes;
          if (rank == 0) mbar_arrive_expect_tx(&full[stage], 2 * kManyStageBytes);  // of both CTAs
          const uint32_t bar = of_first(&full[stage]);
          tma_load_pair(to, &a_map, bar, b * kFp8Block, tile.m * kManyRows + rank * 128, often);
          tma_load_pair(to + 128 * kFp8Block, &w_map, bar, b * kFp8Block, tile.n * kManyCols + rank * 128, often);
        }
        __syncwarp();
        ++issued;
        if (++stage == kManyStages) stage = 0, phase ^= 1;
      }
    }
  } else if (warp < 3) {  // an accumulator each: one waits for its sums while the other issues
    constexpr uint32_t idesc = umma_idesc_f16(kManyRows, kManyCols);
    const uint64_t a0 = umma_smem_desc(smem_addr(smem), 16, 1024, 2);
    const uint64_t w0 = umma_smem_desc(smem_addr(smem) + 128 * kFp8Block, 16, 1024, 2);
    int stage = 0, d = 0;
    uint32_t phase = 0, sums_phase = 1;
    for (int t = pair; rank == 0 && t < tiles && !dead; t += pairs)
      for (int b = 0; b < blocks; ++b) {
        // (what is there earlier first: from the sums' word on there is little to do)
        if (d != warp - 1) {
          if (++stage == kManyStages) stage = 0, phase ^= 1;
          sums_phase ^= d;
          d ^= 1;
          continue;
        }
        const uint64_t a = a0 + stage * (kManyStageBytes >> 4), w = w0 + stage * (kManyStageBytes >> 4);
        const uint32_t to = tmem + d * kManyCols;
        wait_phase(&full[stage], phase, dead, p);
        wait_phase(&sums_empty[d], sums_phase, dead, p);
        dead = agreed(dead);
        if (dead) break;
        tcgen05_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < 4; ++k) umma_e4m3_pair(to, a + 2 * k, w + 2 * k, idesc, k > 0);
          umma_commit_pair(&sums_full[d]);
          umma_commit_pair(&empty[stage]);
        }
        __syncwarp();
        if (++stage == kManyStages) stage = 0, phase ^= 1;
        sums_phase ^= d;
        d ^= 1;
      }
  } else if (warp >= 4) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kMoreRegs));
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    const uint32_t from = tmem + ((uint32_t)(quarter * 32) << 16) + half * 128;
    float* patch = reinterpret_cast<float*>(smem + kManyStages * kManyStageBytes + (warp - 4) * kPatch);
    const uint32_t summed0 = of_first(&sums_empty[0]);
    int d = 0;
    uint32_t phase = 0;
    for (int t = pair; t < tiles && !dead; t += pairs) {
      const Tile tile = tile_of(t, tiles_m, tiles_n);
      const int row = tile.m * kManyRows + rank * 128 + quarter * 32 + lane, col = tile.n * kManyCols + half * 128;
      const float* a_scale = p.a_scales + (long long)min(row, p.m - 1) * blocks;
      const float* w_scale = p.w_scales + (long long)min(col / kFp8Block, (p.n - 1) / kFp8Block) * blocks;
      unsigned long long acc[64];
#pragma unroll
      for (int j = 0; j < 64; ++j) acc[j] = 0;
      // (multiplied when they are needed: not waited for before that)
      float next_a = a_scale[0], next_w = w_scale[0];
      for (int b = 0; b < blocks; ++b) {
        const float scale = next_a * next_w;
        const unsigned long long f = pair_of(scale, scale);
        if (b + 1 < blocks) next_a = a_scale[b + 1], next_w = w_scale[b + 1];
        const uint32_t at = from + d * kManyCols;
        wait_phase(&sums_full[d], phase, dead, p);
        dead = agreed(dead);
        if (dead) break;
        tcgen05_fence_after();
#pragma unroll
        for (int c = 0; c < 128; c += 32) {
          uint32_t v[32];
          tmem_ld16(at + c, v);
          tmem_ld16(at + c + 16, v + 16);
          tmem_ld_wait();
          if (c == 96) {  // all read: the accumulator is free, whatever is still to be added
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) arrive_at(summed0 + d * (uint32_t)sizeof(uint64_t));
          }
#pragma unroll
          for (int j = 0; j < 16; ++j)
            acc[c / 2 + j] = fma2(pair_of(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1])), f, acc[c / 2 + j]);
        }
        phase ^= d;
        d ^= 1;
      }
      if (dead) break;
#pragma unroll
      for (int c = 0; c < 128; c += 32) {
        float v[32];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float2 y = values_of(acc[c / 2 + j]);
          v[2 * j] = y.x, v[2 * j + 1] = y.y;
        }
        store_rows<T>(p, row, col + c, wide, patch, v);
      }
    }
  }
  // After a wait that gave up: what is in flight completes before its memory is given back.
  if (__syncthreads_or(dead)) {
    bool late = false;
    if (warp == 0 && rank == 0)
      for (int s = max(0, issued - kManyStages); s < issued; ++s)
        wait_phase(&full[s % kManyStages], (s / kManyStages) & 1, late, p);
    if ((warp == 1 || warp == 2) && rank == 0) {
      if (elect_one()) umma_commit_pair(&drained);
      __syncwarp();
      wait_phase(&drained, 0, late, p);
    }
    __syncwarp();
    __syncthreads();
  }
  tcgen05_fence_before();
  cluster_sync();  // neither CTA's memory goes while the other may use it
  if (warp == 1) {
    tcgen05_fence_after();
    tmem_dealloc_pair(tmem, 2 * kManyCols);
  }
}

template <class T>
cudaError_t launch_many(const Fp8MatmulParams& p, const Fp8MatmulPlan& plan, const CUtensorMap& a_map,
                        const CUtensorMap& w_map, int sm_count, cudaStream_t st) {
  constexpr int kMaxDevices = 64, smem = kManyStages * kManyStageBytes + 8 * kPatch + 1024;
  static std::atomic<unsigned> asked[kMaxDevices];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const unsigned gen = attr_generation(dev) + 1;
  if (dev >= kMaxDevices || asked[dev].load(std::memory_order_acquire) != gen) {
    if ((e = has_even_regs(fp8_many_kernel<T>)) != cudaSuccess) return e;
    e = cudaFuncSetAttribute(fp8_many_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    if (dev < kMaxDevices) asked[dev].store(gen, std::memory_order_release);
  }
  const int tiles_m = (p.m + kManyRows - 1) / kManyRows, tiles_n = (p.n + kManyCols - 1) / kManyCols;
  const int wide = (reinterpret_cast<uintptr_t>(p.out) | (uintptr_t)(p.out_stride * (long long)sizeof(T))) % 32 == 0;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(2 * fp8_matmul_places(plan, p.m, p.n, sm_count)));
  cfg.blockDim = dim3(kManyThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, fp8_many_kernel<T>, a_map, w_map, p, tiles_m, tiles_n, wide);
}

template <class T>
cudaError_t launch_rows(const Fp8MatmulParams& p, const Fp8MatmulPlan& plan, const CUtensorMap& a_map,
                        const CUtensorMap& w_map, int sm_count, cudaStream_t st) {
  if (plan.rows == kManyRows) return launch_many<T>(p, plan, a_map, w_map, sm_count, st);
  if (plan.cols == 256) return launch_some<T, 256>(p, plan, a_map, w_map, sm_count, st);
  return launch_some<T, 128>(p, plan, a_map, w_map, sm_count, st);
}

}  // namespace

// Up to 64 rows the weight's rows are the product's, and a tile's k is split while a SM has no CTA, or, split already and
// long, has one (us with 1, 2, 4, 8 parts: 1 x 4096 x 14336 12.4, 13.3, 16.4, 22.5; 16 x 4096 x 4096 10.0, 7.6, 6.3, 6.6;
// 16 x 14336 x 4096 27, 17, 14.3, 13.0; 16 x 2048 x 1024 6.2, 5.5, 4.6, 4.4).
// Above, what is expected to take least: a block of k takes a tile of 128 x 128 0.4 us, one of 256 x 256 0.48, tiles go
// round by round over the SMs or their pairs, and a split costs 3 us (128 x 4096 x 4096 15.5, 12.4, 10.0 in tiles of
// 128, 18.0 of 256; 128 x 4096 x 14336 16.9 and 20.2; 256 x 4096 x 14336 29.7 and 20.7).
Fp8MatmulPlan fp8_matmul_plan(int m, int k, int n, int sm_count) {
  const int blocks = (k + kFp8Block - 1) / kFp8Block;
  const long long tiles_n = (n + 127) / 128;
  if (m <= 64) {
    Fp8MatmulPlan plan{m <= 16 ? 16 : m <= 32 ? 32 : 64, 128, 1};
    while (plan.split < kMaxSplit && blocks >= 8 && plan.split * 4 <= blocks &&
           tiles_n * plan.split * 2 <= (plan.split > 1 && plan.split * 16 <= blocks ? 2 : 1) * sm_count)
      plan.split *= 2;
    return plan;
  }
  Fp8MatmulPlan best{};
  double least = 0.0;
  const auto consider = [&](int rows, int cols, int split, int places, double fixed, double block) {
    const long long tiles = (long long)((m + rows - 1) / rows) * ((n + cols - 1) / cols) * split;
    const double us = fixed + (double)((tiles + places - 1) / places) * ((blocks + split - 1) / split) * block;
    if (best.rows == 0 || us < least) least = us, best = {rows, cols, split};
  };
  consider(kManyRows, kManyCols, 1, sm_count / 2, 4.5, 0.48);
  consider(128, 256, 1, sm_count, 3.5, 0.5);
  consider(128, 128, 1, sm_count, 3.0, 0.4);
  for (int split = 2; split <= kMaxSplit / 2 && split * 4 <= blocks; split *= 2)
    if ((m + 127) / 128 * tiles_n * split <= sm_count) consider(128, 128, split, sm_count, 6.0, 0.4);
  return best;
}

int fp8_matmul_places(const Fp8MatmulPlan& plan, int m, int n, int sm_count) {
  const long long parts = (long long)((m + plan.rows - 1) / plan.rows) * ((n + plan.cols - 1) / plan.cols) * plan.split;
  const int most = plan.rows < 128 ? Few<64>::kCtas * sm_count : plan.rows == kManyRows ? sm_count / 2 : sm_count;
  return (int)(plan.split > 1 ? parts : std::min<long long>(parts, most));
}

cudaError_t launch_fp8_matmul(const Fp8MatmulParams& p, const Fp8MatmulPlan& plan, const CUtensorMap& a_map,
                              const CUtensorMap& w_map, int sm_count, cudaStream_t st) {
  if (plan.rows < 128) {
    if (plan.rows == 16) return launch_few<16>(p, plan, a_map, w_map, sm_count, st);
    if (plan.rows == 32) return launch_few<32>(p, plan, a_map, w_map, sm_count, st);
    return launch_few<64>(p, plan, a_map, w_map, sm_count, st);
  }
  if (p.dtype == kTypeF32) return launch_rows<float>(p, plan, a_map, w_map, sm_count, st);
  return p.dtype == kTypeBF16 ? launch_rows<__nv_bfloat16>(p, plan, a_map, w_map, sm_count, st)
                              : launch_rows<__half>(p, plan, a_map, w_map, sm_count, st);
}

}  // namespace tk
