// tk_sample.cu -- a token of each row of logits, from a given random number, after temperature, top-k, top-p and
// min-p.
//
//   w_i = exp((l_i - max) / T);  tokens ranked by (l descending, index ascending)
//   kept: the first top_k of them; of these the shortest prefix with a sum of w of at least top_p times theirs;
//   of these w_i >= min_p.  The token is the first kept one, by index, at which the running sum of w passes
//   random times the sum of all kept.
//
// The answer is a whole number that goes by where one sum passes another, so weights and sums are f64: tokens differ
// from those of exact sums where the random number lies within about 1e-13 of a border, instead of within 1e-7,
// which in a row of 128256 tokens is one row in a hundred.  All sums have a fixed order, or are sums of integers.
//
// A row lies in the shared memory of a cluster's CTAs and is read from memory once.
#include <algorithm>
#include <atomic>

#include "tk_elements.cuh"
#include "tk_internal.h"
#include "tk_kv4.h"
#include "tk_sample.h"

namespace tk {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32, kMaxCluster = 8;
constexpr int kBins = 2048;
constexpr float kNone = -INFINITY;
constexpr double kUnit = 17592186044416.0;  // 2^44: weights as integers, whose sums fit 64 bits

__device__ __forceinline__ void cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Shared memory of the CTA with that rank.
template <class V>
__device__ __forceinline__ V* of_rank(V* mine, int rank) {
  uint64_t at;
  asm("mapa.u64 %0, %1, %2;" : "=l"(at) : "l"(reinterpret_cast<uint64_t>(mine)), "r"(rank));
  return reinterpret_cast<V*>(at);
}

// Order of values as that of whole numbers.
template <class T>
struct Key;
template <>
struct Key<float> {
  static constexpr int kBits = 32;
};
template <>
struct Key<__half> {
  static constexpr int kBits = 16;
};
template <>
struct Key<__nv_bfloat16> {
  static constexpr int kBits = 16;
};
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t b = __float_as_uint(v);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint32_t key_of(__half v) {
  const uint32_t b = __half_as_ushort(v);
  return (b & 0x8000u ? ~b : b | 0x8000u) & 0xffffu;
}
__device__ __forceinline__ uint32_t key_of(__nv_bfloat16 v) {
  const uint32_t b = __bfloat16_as_ushort(v);
  return (b & 0x8000u ? ~b : b | 0x8000u) & 0xffffu;
}

struct Shared {
  uint32_t count[kBins];
  unsigned long long mass[kBins];
  // read by the other CTAs
  double warp_sum[kWarps];
  int warp_count[kWarps];
  float warp_max[kWarps];
  // written by another CTA
  int index;
  // own
  double all_sum[kMaxCluster * kWarps];
  int all_count[kMaxCluster * kWarps];
  double scan[kWarps];
  unsigned long long scan_mass[kWarps];
  uint32_t scan_count[kWarps];
  uint32_t bin;
  unsigned long long above_mass;
  uint32_t above_count, bin_count;
  unsigned long long bin_mass;
};

// Where the kept ones end: all of a key above, and the first `ties` of that key.
struct Cut {
  uint32_t key;
  unsigned long long ties, equal;  // kept of, and all with that key
  unsigned long long mass;         // of the kept ones
};

template <class T>
__global__ void __launch_bounds__(kThreads) sample_tokens_kernel(SampleParams p, int cluster, int slice) {
  extern __shared__ __align__(16) uint8_t dynamic[];
  Shared& sh = *reinterpret_cast<Shared*>(dynamic);
  T* mine = reinterpret_cast<T*>(dynamic + (sizeof(Shared) + 15) / 16 * 16);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = blockIdx.x % cluster;
  const long long row = blockIdx.x / cluster;
  const int first = rank * slice, n = max(0, min(slice, p.vocab - first));
  after_previous();
  const T* src = static_cast<const T*>(p.logits) + row * p.stride + first;

  // The row into shared memory: NaN as -inf, -0 as 0; its largest, and how many there are.
  float most = kNone;
  int valid = 0;
  auto take = [&](int i, float v) {
    v = v != v ? kNone : v + 0.f;
    mine[i] = from_f32<T>(v);
    most = fmaxf(most, v);
    valid += v > kNone;
  };
  constexpr int kVec = 16 / sizeof(T);
  if (reinterpret_cast<uintptr_t>(src) % 16 == 0) {
    const int vecs = n / kVec;
    for (int i = tid; i < vecs; i += kThreads) {
      const uint4 raw = reinterpret_cast<const uint4*>(src)[i];
      const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int j = 0; j < kVec; ++j) take(i * kVec + j, to_f32(e[j]));
    }
    for (int i = vecs * kVec + tid; i < n; i += kThreads) take(i, to_f32(src[i]));
  } else {
    for (int i = tid; i < n; i += kThreads) take(i, to_f32(src[i]));
  }
#pragma unroll
  for (int off = 16; off; off >>= 1) {
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, off));
    valid += __shfl_xor_sync(0xffffffffu, valid, off);
  }
  if (lane == 0) sh.warp_max[warp] = most, sh.warp_count[warp] = valid;
  cluster_sync();
  most = kNone;
  valid = 0;
  for (int i = lane; i < cluster * kWarps; i += 32) {
    most = fmaxf(most, of_rank(sh.warp_max, i / kWarps)[i % kWarps]);
    valid += of_rank(sh.warp_count, i / kWarps)[i % kWarps];
  }
#pragma unroll
  for (int off = 16; off; off >>= 1) {
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, off));
    valid += __shfl_xor_sync(0xffffffffu, valid, off);
  }
  cluster_sync();  // warp_max and warp_count are free again

  const float heat = p.temperature ? p.temperature[row] : 1.f;
  const bool greedy = !(heat > 0.f);
  const double slope = greedy ? 0.0 : 1.4426950408889634 / (double)heat;  // log2 e / T
  const bool endless = most == INFINITY;
  // log2 of a weight; what is not there is at -inf.  Where the largest is infinite only its equals are there.
  auto exponent = [&](float l) -> double {
    if (l == most) return 0.0;
    if (endless || l == kNone) return -INFINITY;
    return ((double)l - (double)most) * slope;
  };
  auto weight = [&](double t) -> double { return t < -1022.0 ? 0.0 : exp2(t); };
  auto value = [&](int i) -> float { return to_f32(mine[i]); };

  // By descending digits of the keys: the cut after `wanted` tokens, or after a sum of `wanted`.
  auto cut_at = [&](bool by_mass, unsigned long long wanted, bool masses) -> Cut {
    Cut cut{0, 0, 0, 0};
    uint32_t known = 0;
    unsigned long long above = 0, above_mass = 0, equal_mass = 0;
    constexpr int kBits = Key<T>::kBits;
    for (int high = kBits; high > 0;) {
      const int digit = min(11, high), shift = high - digit;
      for (int i = tid; i < kBins; i += kThreads) sh.count[i] = 0, sh.mass[i] = 0;
      __syncthreads();
      for (int i = tid; i < n; i += kThreads) {
        const float l = value(i);
        const uint32_t key = key_of(mine[i]);
        if (l > kNone && (key & known) == cut.key) {
          const uint32_t bin = key >> shift & ((1u << digit) - 1u);
          atomicAdd(&sh.count[bin], 1u);
          if (masses) atomicAdd(&sh.mass[bin], (unsigned long long)(weight(exponent(l)) * kUnit + 0.5));
        }
      }
      cluster_sync();
      // thread t sums four bins over the CTAs, from the top down
      constexpr int kEach = kBins / kThreads;
      uint32_t c[kEach], my_count = 0;
      unsigned long long m[kEach], my_mass = 0;
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        const int bin = kBins - 1 - (tid * kEach + j);
        c[j] = 0, m[j] = 0;
        for (int r = 0; r < cluster; ++r) c[j] += of_rank(sh.count, r)[bin], m[j] += of_rank(sh.mass, r)[bin];
        my_count += c[j], my_mass += m[j];
      }
      uint32_t inc = my_count;
      unsigned long long inc_mass = my_mass;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const uint32_t o = __shfl_up_sync(0xffffffffu, inc, off);
        const unsigned long long om = __shfl_up_sync(0xffffffffu, inc_mass, off);
        if (lane >= off) inc += o, inc_mass += om;
      }
      if (lane == 31) sh.scan_count[warp] = inc, sh.scan_mass[warp] = inc_mass;
      __syncthreads();
      unsigned long long at = above + inc - my_count, at_mass = above_mass + inc_mass - my_mass;
      for (int w = 0; w < warp; ++w) at += sh.scan_count[w], at_mass += sh.scan_mass[w];
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        const bool here = by_mass ? at_mass < wanted && wanted <= at_mass + m[j] : at < wanted && wanted <= at + c[j];
        if (here) {
          sh.bin = kBins - 1 - (tid * kEach + j);
          sh.above_count = (uint32_t)at, sh.above_mass = at_mass;
          sh.bin_count = c[j], sh.bin_mass = m[j];
        }
        at += c[j], at_mass += m[j];
      }
      cluster_sync();
      above = sh.above_count, above_mass = sh.above_mass;
      cut.equal = sh.bin_count, equal_mass = sh.bin_mass;
      cut.key |= sh.bin << shift;
      known |= ((1u << digit) - 1u) << shift;
      high = shift;
      __syncthreads();
    }
    const unsigned long long each = equal_mass / cut.equal;
    if (!by_mass)
      cut.ties = wanted - above;
    else
      cut.ties = each ? min(cut.equal, (wanted - above_mass + each - 1) / each) : cut.equal;
    cut.mass = above_mass + cut.ties * each;
    return cut;
  };

  if (most == kNone) {
    if (rank == 0 && tid == 0) {
      p.tokens[row] = -1;
      if (p.kept) p.kept[row] = 0;
    }
    cluster_sync();
    return;
  }
  const int k = greedy || !p.top_k ? 0 : p.top_k[row];
  const float top_p = greedy || !p.top_p ? 1.f : p.top_p[row];
  const float min_p = greedy || !p.min_p ? 0.f : p.min_p[row];
  Cut cut{0, 0, 0, 0};
  const uint32_t top_key = key_of(from_f32<T>(most));
  if (greedy) {
    cut.key = top_key, cut.ties = 1, cut.equal = 2;
  } else {
    const bool by_k = k > 0 && k < valid, by_p = top_p < 1.f;
    if (by_k) cut = cut_at(false, (unsigned long long)k, by_p);
    if (by_p) {
      unsigned long long base = cut.mass;
      if (!by_k) {  // the sum of all
        unsigned long long sum = 0;
        for (int i = tid; i < n; i += kThreads) sum += (unsigned long long)(weight(exponent(value(i))) * kUnit + 0.5);
#pragma unroll
        for (int off = 16; off; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        if (lane == 0) sh.mass[warp] = sum;
        cluster_sync();
        base = 0;
        for (int i = 0; i < cluster * kWarps; ++i) base += of_rank(sh.mass, i / kWarps)[i % kWarps];
        cluster_sync();
      }
      const double share = (double)fmaxf(top_p, 0.f) * (double)base;
      const unsigned long long wanted = (unsigned long long)share;
      cut = cut_at(true, max(1ull, min(base, wanted + ((double)wanted < share))), true);
    }
  }
  const double least = min_p > 0.f ? (double)fminf(min_p, 1.f) : 0.0;

  // Warps own runs of the row, so that the runs' sums stand in the order of the tokens.
  const int run = (slice + kWarps * 32 - 1) / (kWarps * 32) * 32;
  const int r0 = min(n, warp * run), r1 = min(n, r0 + run);
  // The first kept ones of a key, by index.
  int last = 0x7fffffff;
  if (cut.ties < cut.equal) {
    int equal = 0;
    for (int i = r0 + lane; i < r1; i += 32) equal += key_of(mine[i]) == cut.key;
#pragma unroll
    for (int off = 16; off; off >>= 1) equal += __shfl_xor_sync(0xffffffffu, equal, off);
    if (lane == 0) sh.warp_count[warp] = equal;
    cluster_sync();
    unsigned long long before = 0;
    for (int i = 0; i < rank * kWarps + warp; ++i) before += of_rank(sh.warp_count, i / kWarps)[i % kWarps];
    if (before < cut.ties && cut.ties <= before + equal) {
      for (int i0 = r0; i0 < r1; i0 += 32) {
        const bool is = i0 + lane < r1 && key_of(mine[i0 + lane]) == cut.key;
        const uint32_t votes = __ballot_sync(0xffffffffu, is);
        if (before + __popc(votes) >= cut.ties) {
          const int nth = (int)(cut.ties - before);
          if (is && __popc(votes & (0xffffffffu >> (31 - lane))) == nth)
            for (int r = 0; r < cluster; ++r) *of_rank(&sh.index, r) = first + i0 + lane;
          break;
        }
        before += __popc(votes);
      }
    }
    cluster_sync();
    last = sh.index;
  }
  // 0 where the token is not kept
  auto kept_weight = [&](int i, bool& is) -> double {
    const float l = value(i);
    const uint32_t key = key_of(mine[i]);
    is = l > kNone && (!endless || l == most) && (key > cut.key || (key == cut.key && first + i <= last));
    if (!is) return 0.0;
    const double w = weight(exponent(l));
    is = w >= least;
    return is ? w : 0.0;
  };
  double sum = 0.0;
  int count = 0;
  for (int i = r0 + lane; i < r1; i += 32) {
    bool is;
    sum += kept_weight(i, is);
    count += is;
  }
#pragma unroll
  for (int off = 16; off; off >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, off);
    count += __shfl_xor_sync(0xffffffffu, count, off);
  }
  __syncthreads();
  if (lane == 0) sh.warp_sum[warp] = sum, sh.warp_count[warp] = count;
  cluster_sync();
  for (int i = tid; i < cluster * kWarps; i += kThreads) {
    sh.all_sum[i] = of_rank(sh.warp_sum, i / kWarps)[i % kWarps];
    sh.all_count[i] = of_rank(sh.warp_count, i / kWarps)[i % kWarps];
  }
  cluster_sync();  // no CTA reads another's after this
  double total = 0.0;
  int all = 0;
  for (int i = 0; i < cluster * kWarps; ++i) total += sh.all_sum[i], all += sh.all_count[i];
  if (rank == 0 && tid == 0 && p.kept) p.kept[row] = all;
  const float u = p.random[row];
  const double goal = (u > 0.f ? (double)fminf(u, 1.f) : 0.0) * total;
  // the run in which the sum passes the goal; the last with a sum where rounding keeps it from that
  double before = 0.0, at = 0.0;
  int owner = -1;
  for (int i = 0; i < cluster * kWarps; ++i) {
    const double s = sh.all_sum[i];
    if (s > 0.0) {
      owner = i, before = at;
      if (at + s > goal) break;
    }
    at += s;
  }
  if (owner / kWarps != rank) return;
  // All threads on that run, consecutive tokens each.
  const int w0 = min(n, owner % kWarps * run), w1 = min(n, w0 + run), each = (run + kThreads - 1) / kThreads;
  const int i0 = min(w1, w0 + tid * each), i1 = min(w1, i0 + each);
  double part = 0.0;
  bool is;
  for (int i = i0; i < i1; ++i) part += kept_weight(i, is);
  double inc = part;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const double o = __shfl_up_sync(0xffffffffu, inc, off);
    if (lane >= off) inc += o;
  }
  if (lane == 31) sh.scan[warp] = inc;
  if (tid == 0) sh.index = -1, sh.bin = 0;
  __syncthreads();
  for (int w = 0; w < warp; ++w) before += sh.scan[w];
  // the first thread whose end passes the goal, or the last with a sum
  const double lo = before + inc - part;
  const bool passes = part > 0.0 && before + inc > goal;
  if (passes) atomicMax(&sh.bin, (uint32_t)(kThreads - tid));
  if (part > 0.0) atomicMax(&sh.index, tid);
  __syncthreads();
  const int winner = sh.bin ? kThreads - (int)sh.bin : sh.index;
  if (tid == winner) {
    double running = lo;
    int token = -1;
    for (int i = i0; i < i1; ++i) {
      const double w = kept_weight(i, is);
      if (w > 0.0) {
        token = first + i;
        running += w;
        if (running > goal) break;
      }
    }
    p.tokens[row] = token;
  }
}

template <class T>
cudaError_t launch_sample(const SampleParams& p, int sm_count, cudaStream_t st) {
  constexpr int kMaxDevices = 64, kHead = (sizeof(Shared) + 15) / 16 * 16, kMaxBytes = 227 * 1024;
  static std::atomic<unsigned> asked[kMaxDevices];
  int cluster = 1;
  while (cluster < kMaxCluster && ((long long)p.rows * cluster * 2 <= sm_count ||
                                   kHead + ((p.vocab + cluster - 1) / cluster + 8) * (int)sizeof(T) > kMaxBytes))
    cluster *= 2;
  const int slice = ((p.vocab + cluster - 1) / cluster + 7) / 8 * 8, smem = kHead + slice * (int)sizeof(T);
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const unsigned gen = attr_generation(dev) + 1;
  if (dev >= kMaxDevices || asked[dev].load(std::memory_order_acquire) != gen) {
    e = cudaFuncSetAttribute(sample_tokens_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxBytes);
    if (e != cudaSuccess) return e;
    if (dev < kMaxDevices) asked[dev].store(gen, std::memory_order_release);
  }
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(p.rows * cluster));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, sample_tokens_kernel<T>, p, cluster, slice);
}

}  // namespace

cudaError_t launch_sample_tokens(const SampleParams& p, int dtype, int sm_count, cudaStream_t st) {
  if (dtype == kTypeF32) return launch_sample<float>(p, sm_count, st);
  return dtype == kTypeBF16 ? launch_sample<__nv_bfloat16>(p, sm_count, st) : launch_sample<__half>(p, sm_count, st);
}

}  // namespace tk
