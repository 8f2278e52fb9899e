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

// Waits for the phase of `bar`; gives up, for good, after timeout_ns.  The timer is read once in many tries, since a read
// takes longer than a phase should be noticed late, and the phase is looked at once more after the last read: lanes of a
// warp that wait for one phase agree.
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
// The weight's rows are the product's 128 rows, the activations its NT columns.  The CTAs of a cluster share a
// tile's blocks of k and add their sums through shared memory, in the order of their ranks.

constexpr int kFewThreads = 192;  // a warp of copies, one of products, four of sums
constexpr int kMaxStages = 8, kMaxSplit = 8;

template <int NT>
struct Few {
  static constexpr int kStep = NT == 128 ? 1 : 2;  // blocks of k between two waits
  static constexpr int kBlockBytes = (128 + NT) * kFp8Block, kStageBytes = kStep * kBlockBytes;
  static constexpr uint32_t kColumns = 2 * kStep * NT;  // of tensor memory: two steps
};

template <int NT>
__global__ void __launch_bounds__(kFewThreads) fp8_few_kernel(const __grid_constant__ CUtensorMap a_map,
                                                              const __grid_constant__ CUtensorMap w_map,
                                                              Fp8MatmulParams p, int split, int stages) {
  using M = Few<NT>;
  constexpr int KS = M::kStep;
  extern __shared__ uint8_t dynamic[];
  __shared__ uint64_t full[kMaxStages], empty[kMaxStages], sums_full[2], sums_empty[2], drained;
  __shared__ uint32_t tmem_slot;
  __shared__ __align__(16) float factors[4][2][KS][NT];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* smem = dynamic + ((1024u - (smem_addr(dynamic) & 1023u)) & 1023u);
  const int tile = blockIdx.x / split, rank = blockIdx.x % split, token0 = blockIdx.y * NT;
  const int blocks = (p.k + kFp8Block - 1) / kFp8Block;
  const int b0 = (int)((long long)blocks * rank / split), b1 = (int)((long long)blocks * (rank + 1) / split);
  const int steps = (b1 - b0 + KS - 1) / KS;
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) mbar_init(&full[s], 1), mbar_init(&empty[s], 1);
    for (int s = 0; s < 2; ++s) mbar_init(&sums_full[s], 1), mbar_init(&sums_empty[s], 4);
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
  unsigned long long acc[NT / 2];
  if (warp == 0) {
    const uint64_t once = l2_evict_first(), often = l2_evict_last();
    for (int s = 0; s < steps; ++s) {
      const int stage = s % stages;
      if (s >= stages) wait_phase(&empty[stage], (s / stages - 1) & 1, dead, p);
      if (__any_sync(0xffffffffu, dead)) {
        dead = true;
        break;
      }
      const int n = min(KS, b1 - b0 - s * KS);
      if (elect_one()) {
        uint8_t* to = smem + stage * M::kStageBytes;
        mbar_arrive_expect_tx(&full[stage], n * M::kBlockBytes);
        for (int i = 0; i < n; ++i) {
          const int x = (b0 + s * KS + i) * kFp8Block;
          tma_load_2d(to + i * 16384, &w_map, &full[stage], x, tile * 128, once);
          tma_load_2d(to + KS * 16384 + i * NT * kFp8Block, &a_map, &full[stage], x, token0, often);
        }
      }
      __syncwarp();
      issued = s + 1;
    }
  } else if (warp == 1) {
    constexpr uint32_t idesc = umma_idesc_f16(128, NT);
    for (int s = 0; s < steps; ++s) {
      const int stage = s % stages, d = s & 1;
      if (s >= 2) wait_phase(&sums_empty[d], (s / 2 - 1) & 1, dead, p);
      wait_phase(&full[stage], (s / stages) & 1, dead, p);
      if (__any_sync(0xffffffffu, dead)) {
        dead = true;
        break;
      }
      tcgen05_fence_after();
      const int n = min(KS, b1 - b0 - s * KS);
      if (elect_one()) {
        const uint32_t at = smem_addr(smem) + stage * M::kStageBytes;
        for (int i = 0; i < n; ++i) {
          const uint64_t w = umma_smem_desc(at + i * 16384, 16, 1024, 2);
          const uint64_t a = umma_smem_desc(at + KS * 16384 + i * NT * kFp8Block, 16, 1024, 2);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_e4m3(tmem + (d * KS + i) * NT, w + 2 * k, a + 2 * k, idesc, k > 0);
        }
        umma_commit(&empty[stage]);
        umma_commit(&sums_full[d]);
      }
      __syncwarp();
    }
  } else {
    const int quarter = warp & 3, at = warp - 2;
    const uint32_t from = tmem + ((uint32_t)(quarter * 32) << 16);
#pragma unroll
    for (int j = 0; j < NT / 2; ++j) acc[j] = 0;
    constexpr int kEach = (NT + 31) / 32;
    float next[KS][kEach], next_w[KS];  // multiplied when they are needed: not waited for before that
    auto fetch = [&](int s) {
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        const int b = b0 + s * KS + i;
        next_w[i] = b < b1 ? p.w_scales[(long long)tile * blocks + b] : 0.f;
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
          const int j = e * 32 + lane, token = token0 + j;
          next[i][e] = b < b1 && j < NT && token < p.m ? p.a_scales[(long long)token * blocks + b] : 0.f;
        }
      }
    };
    fetch(0);
    for (int s = 0; s < steps; ++s) {
      const int d = s & 1;
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int e = 0; e < kEach; ++e)
          if (e * 32 + lane < NT) factors[at][d][i][e * 32 + lane] = next[i][e] * next_w[i];
      if (s + 1 < steps) fetch(s + 1);
      __syncwarp();
      wait_phase(&sums_full[d], (s / 2) & 1, dead, p);
      if (__any_sync(0xffffffffu, dead)) {
        dead = true;
        break;
      }
      tcgen05_fence_after();
      const int n = min(KS, b1 - b0 - s * KS);
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        if (i >= n) break;
#pragma unroll
        for (int c = 0; c < NT; c += 16) {
          uint32_t t[16];
          tmem_ld16(from + (d * KS + i) * NT + c, t);
          tmem_ld_wait();
          const float4* f = reinterpret_cast<const float4*>(&factors[at][d][i][c]);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float4 g = f[j];
            unsigned long long* to = &acc[c / 2 + 2 * j];
            to[0] = fma2(pair_of(__uint_as_float(t[4 * j]), __uint_as_float(t[4 * j + 1])), pair_of(g.x, g.y), to[0]);
            to[1] = fma2(pair_of(__uint_as_float(t[4 * j + 2]), __uint_as_float(t[4 * j + 3])), pair_of(g.z, g.w), to[1]);
          }
        }
      }
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sums_empty[d]);
    }
  }
  // After a wait that gave up: what is in flight completes before its memory is given back.
  if (__syncthreads_or(dead)) {
    bool late = false;
    if (warp == 0)
      for (int s = max(0, issued - stages); s < issued; ++s) wait_phase(&full[s % stages], (s / stages) & 1, late, p);
    if (warp == 1) {
      if (elect_one()) umma_commit(&drained);
      __syncwarp();
      wait_phase(&drained, 0, late, p);
    }
    dead = true;
    __syncthreads();
  }
  const int row = (warp & 3) * 32 + lane, out_row = tile * 128 + row;
  if (split == 1) {
    if (warp >= 2 && !dead && out_row < p.n) {
#pragma unroll
      for (int j = 0; j < NT / 2; ++j) {
        const float2 v = values_of(acc[j]);
        const int token = token0 + 2 * j;
        if (token < p.m) store_out(p, token * p.out_stride + out_row, v.x);
        if (token + 1 < p.m) store_out(p, (token + 1) * p.out_stride + out_row, v.y);
      }
    }
  } else {
    float* mine = reinterpret_cast<float*>(smem);  // [NT][128]
    if (warp >= 2) {
#pragma unroll
      for (int j = 0; j < NT / 2; ++j) {
        const float2 v = values_of(acc[j]);
        mine[2 * j * 128 + row] = v.x;
        mine[(2 * j + 1) * 128 + row] = v.y;
      }
    }
    cluster_sync();
    // the tokens' columns over the CTAs, four rows a thread, all CTAs' values at once
    const int tokens = min(NT, p.m - token0), j0 = tokens * rank / split, j1 = tokens * (rank + 1) / split;
    for (int i = threadIdx.x; !dead && i < (j1 - j0) * 32; i += kFewThreads) {
      const int j = j0 + i / 32, row4 = i % 32 * 4, n = tile * 128 + row4;
      if (n >= p.n) continue;
      const uint32_t from = smem_addr(mine + j * 128 + row4);
      float4 v[kMaxSplit];
#pragma unroll
      for (int r = 0; r < kMaxSplit; ++r)
        if (r < split) v[r] = ld_peer(from, r);
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int r = 0; r < kMaxSplit; ++r)
        if (r < split) sum.x += v[r].x, sum.y += v[r].y, sum.z += v[r].z, sum.w += v[r].w;
      store_four(p, (token0 + j) * p.out_stride + n, p.n - n, sum);
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
                       const CUtensorMap& w_map, cudaStream_t st) {
  using M = Few<NT>;
  constexpr int kMaxDevices = 64;
  static std::atomic<unsigned> asked[kMaxDevices];
  const int stages = std::min(kMaxStages, (NT <= 32 ? 112 * 1024 : 222 * 1024) / M::kStageBytes);
  const int smem = std::max(stages * M::kStageBytes, NT * 512) + 1024;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const unsigned gen = attr_generation(dev) + 1;
  if (dev >= kMaxDevices || asked[dev].load(std::memory_order_acquire) != gen) {
    e = cudaFuncSetAttribute(fp8_few_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
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
  cfg.gridDim = dim3((unsigned)((p.n + 127) / 128 * plan.split), (unsigned)((p.m + NT - 1) / NT));
  cfg.blockDim = dim3(kFewThreads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = plan.split > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, fp8_few_kernel<NT>, a_map, w_map, p, plan.split, stages);
}

// ---- many rows -----------------------------------------------------------------------------------------
//
// The activations are the product's rows, 256 rows of the weight its columns.  Two CTAs share a product of 256 x 256:
// each brings its 128 rows and half of the columns' weight, and has its rows' sums in its tensor memory.  (Alone, a
// CTA would bring 48 KB a block to its 128 x 256 products, and writing and reading them would take shared memory
// longer than the products take.)  A thread adds half of a row in registers, so that its scale is one number a block:
// sum += scale * product.  Two accumulators of 256 columns fill tensor memory: one is added up while the other's
// products run.  Pairs of CTAs walk over the tiles.

// A warpgroup with a warp of copies and two of products, two warpgroups of sums.  A thread of the sums holds 128 of them: the
// registers of the launch, 168 for each thread, are handed from the first group to the others, 40 and 2 x 232 of 3 x 168.
constexpr int kManyThreads = 384, kManyRegs = 168, kManyFewRegs = 40, kManyMoreRegs = 232;
static_assert(kManyFewRegs + 2 * kManyMoreRegs <= 3 * kManyRegs, "the groups' shares");
constexpr int kManyRows = 256, kManyCols = 256, kManyStages = 6, kManyStageBytes = 2 * 128 * kFp8Block;  // a CTA's part
constexpr int kManyGroup = 8;  // tiles of rows that share the weight's tiles at a time, for L2
constexpr int kPatch = 32 * 33 * 4;  // bytes of a warp's corner of shared memory, for rows off their 32-byte boundary

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

struct ManyTile {
  int m, n;
};
__device__ __forceinline__ ManyTile many_tile(int t, int tiles_m, int tiles_n) {
  const int group = t / (kManyGroup * tiles_n), first = group * kManyGroup, rows = min(kManyGroup, tiles_m - first);
  const int r = t - group * kManyGroup * tiles_n;
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
  if (warp < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kManyFewRegs));
  if (warp == 0) {
    const uint64_t often = l2_evict_last();
    int stage = 0;
    uint32_t phase = 1;  // a barrier's phase before its first counts as complete
    for (int t = pair; t < tiles && !dead; t += pairs) {
      const ManyTile tile = many_tile(t, tiles_m, tiles_n);
      for (int b = 0; b < blocks; ++b) {
        wait_phase(&empty[stage], phase, dead, p);
        __syncwarp();
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
        __syncwarp();
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
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kManyMoreRegs));
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    const uint32_t from = tmem + ((uint32_t)(quarter * 32) << 16) + half * 128;
    float* patch = reinterpret_cast<float*>(smem + kManyStages * kManyStageBytes + (warp - 4) * kPatch);
    const uint32_t summed0 = of_first(&sums_empty[0]);
    int d = 0;
    uint32_t phase = 0;
    for (int t = pair; t < tiles && !dead; t += pairs) {
      const ManyTile tile = many_tile(t, tiles_m, tiles_n);
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
        __syncwarp();
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
      T* out = static_cast<T*>(p.out) + row * p.out_stride + col;
#pragma unroll
      for (int c = 0; c < 128; c += 32) {
        float v[32];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float2 y = values_of(acc[c / 2 + j]);
          v[2 * j] = y.x, v[2 * j + 1] = y.y;
        }
        if (wide && col + c + 32 <= p.n) {
          if (row < p.m) store_32(out + c, v);
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) patch[lane * 33 + j] = v[j];
          __syncwarp();
          const int rows = min(32, p.m - (row - lane));
          T* corner = static_cast<T*>(p.out) + (long long)(row - lane) * p.out_stride + col + c + lane;
          if (col + c + lane < p.n)
            for (int r = 0; r < rows; ++r) corner[r * p.out_stride] = from_f32<T>(patch[r * 33 + lane]);
          __syncwarp();
        }
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
cudaError_t launch_many(const Fp8MatmulParams& p, const CUtensorMap& a_map, const CUtensorMap& w_map, int sm_count,
                        cudaStream_t st) {
  constexpr int kMaxDevices = 64, smem = kManyStages * kManyStageBytes + 8 * kPatch + 1024;
  static std::atomic<unsigned> asked[kMaxDevices];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const unsigned gen = attr_generation(dev) + 1;
  if (dev >= kMaxDevices || asked[dev].load(std::memory_order_acquire) != gen) {
    cudaFuncAttributes has{};
    if ((e = cudaFuncGetAttributes(&has, fp8_many_kernel<T>)) != cudaSuccess) return e;
    if (has.numRegs < kManyRegs) return cudaErrorInvalidKernelImage;  // the sums would wait for registers for good
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
  cfg.gridDim = dim3((unsigned)(2 * std::min(sm_count / 2, tiles_m * tiles_n)));
  cfg.blockDim = dim3(kManyThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, fp8_many_kernel<T>, a_map, w_map, p, tiles_m, tiles_n, wide);
}

}  // namespace

Fp8MatmulPlan fp8_matmul_plan(int m, int k, int n, int sm_count) {
  Fp8MatmulPlan plan;
  if (m > 256) return {kManyCols, 1};
  plan.tile = m <= 16 ? 16 : m <= 32 ? 32 : m <= 64 ? 64 : 128;
  const long long tiles = (long long)((n + 127) / 128) * ((m + plan.tile - 1) / plan.tile);
  const int blocks = (k + kFp8Block - 1) / kFp8Block;
  plan.split = 1;
  while (plan.split < 8 && tiles * plan.split * 2 <= sm_count * 2 && plan.split * 4 <= blocks) plan.split *= 2;
  return plan;
}

void fp8_box_rows(const Fp8MatmulPlan& plan, int* a_rows, int* w_rows) {
  *a_rows = std::min(plan.tile, 128);
  *w_rows = 128;
}

cudaError_t launch_fp8_matmul(const Fp8MatmulParams& p, const Fp8MatmulPlan& plan, const CUtensorMap& a_map,
                              const CUtensorMap& w_map, int sm_count, cudaStream_t st) {
  if (plan.tile == kManyCols) {
    if (p.dtype == kTypeF32) return launch_many<float>(p, a_map, w_map, sm_count, st);
    return p.dtype == kTypeBF16 ? launch_many<__nv_bfloat16>(p, a_map, w_map, sm_count, st)
                                : launch_many<__half>(p, a_map, w_map, sm_count, st);
  }
  if (plan.tile == 16) return launch_few<16>(p, plan, a_map, w_map, st);
  if (plan.tile == 32) return launch_few<32>(p, plan, a_map, w_map, st);
  if (plan.tile == 64) return launch_few<64>(p, plan, a_map, w_map, st);
  return launch_few<128>(p, plan, a_map, w_map, st);
}

}  // namespace tk
