// tk_sample.cu -- a token of each row of logits, from a given random number, after temperature, top-k, top-p and
// min-p.
//
//   w_i = exp((l_i - max) / T);  tokens ranked by (l descending, index ascending)
//   kept: the first top_k of them; of these the shortest prefix with a sum of w of at least top_p times theirs;
//   of these w_i >= min_p.  The token is the first kept one, by index, at which the running sum of w passes
//   random times the sum of all kept.
//
// The answer is a whole number that goes by where one sum passes another, so weights and sums are f64: a token differs
// from that of exact sums where the random number lies within about 1e-13 of a border, instead of within 1e-7,
// which in a row of 128256 tokens is one row in a hundred.  All sums have a fixed order, or are sums of integers: in units of
// their bin, so that a goal among 128255 tokens of a weight of 2^-39 is found to the token.
//
// A row lies in the shared memory of a cluster's CTAs and is read from memory once.  Then, by what the row asks for:
//   top-k (few)       a level that at least top_k tokens reach, from the threads' largest; those tokens, some twice
//                     top_k, are sorted by one CTA, which does the rest on its own
//   top-p             the same with a list of some 200 to 400, where these are likely to hold the sum; otherwise sums of w by
//                     64ths of an octave of w, then a pass with exact sums in which the tokens of the part where the sum
//                     passes its goal are listed; those are sorted
//   either, with more equal values than a list holds, or many top-k: the keys' digits one after the other
// and, where that pass has not done it, a last one with the sums of what is kept.
//
// Bound by the passes' instructions (plain f32 rows: 67 a token in all, of which the weight is some 25, half of them f64; ALU the
// busiest pipe at 45 %, issue slots 62 % busy) and, of a row, by the steps between them, which wait for one another:
// barriers of a cluster at 0.7 us, a sort at 4.  us: 1 x 128256 f32, all filters, 11 over the same logits, 14 from memory; a
// row alone whose top-p keeps half of its tokens 25; 64 x 128256 bf16, plain 23.5, top-k 16, flat rows with top-p 61, a
// mixture 43.6; 256 x 32000 f32, plain 28.3.  Rows off their 16-byte boundary are read by elements: 64 x 50257 bf16 13.2, plain,
// 33.8, mixed, and 50256 12.5 and 32.5.  (CTAs of 256 threads are not faster, nor is the entry of a list found by
// parts of its range instead of by sorting it: equal values meet in one counter.)
#include <algorithm>
#include <atomic>

#include "tk_elements.cuh"
#include "tk_internal.h"
#include "tk_kv4.h"
#include "tk_sample.h"

namespace tk {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32, kMaxCluster = 8, kMaxWarps = kMaxCluster * kWarps;
constexpr int kBins = 2048, kList = 1024, kPer = kList / kThreads, kFew = 400, kReach = 192;
constexpr int kParts = 512;  // of an octave of weights, in the table
constexpr float kBinUnit = 65536.f;  // of a bin's sum: its largest weight
constexpr int kMostBytes = 112 * 1024;  // of a CTA, unless no cluster is large enough for that
constexpr float kNone = -INFINITY, kHuge = 3.4028235e38f;
// Weights of one bin as whole numbers, whose sums are the same in any order: in a list, and among any number of tokens, the bin's
// largest has up to 2^51 and 2^44 units, so that 64 bits hold the sums.
constexpr int kListBits = 51, kRowBits = 44;
constexpr double kWhole = 4503599627370496.0, kRound = 1.5 * kWhole;  // 2^52: added, a value's units are whole

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

// Order of values as that of whole numbers; 16-bit types have keys of 16 bits.
template <class T>
constexpr int kKeyBits = sizeof(T) * 8;
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

// What ranks need.
struct Ranked {
  union {
    struct {
      union {
        uint32_t sums[kBins];
        unsigned long long sorted[2][kList];  // (key, ~index) of all CTAs' lists
      };
      unsigned long long list[kList];  // found here
    };
    struct {
      uint32_t count[kBins];
      unsigned long long mass[kBins];
    } digits;
  };
};
struct Shared {
  double table[kParts];  // 2^(i / kParts)
  // of all CTAs' warps, written by each into every CTA's
  double all_sum[kMaxWarps], all_head[kMaxWarps], all_mass[kMaxWarps];
  float all_most[kMaxWarps], all_level[kMaxWarps], all_few[kMaxWarps], all_sample[kMaxWarps];
  int all_equal[kMaxWarps], all_count[kMaxWarps];
  int all_listed[kMaxCluster];
  uint32_t cut_key;
  int cut_index;
  // own
  double rest;  // of the goal, for that bin
  int rest_bin;
  int listed, first_equal;
  unsigned long long extra[kWarps];
  int extra_count[kWarps];
  float level[kMaxWarps / 32];
  double scan[kWarps];
  unsigned long long scan_mass[kWarps];
  uint32_t bin;
  unsigned long long above_mass;
  uint32_t bin_count;
  unsigned long long bin_mass;
  int long_rows[kWarps], chosen;
};

// Sums of all threads before this one, and of all.
__device__ __forceinline__ double scan_threads(double v, double* part, double* total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  double inc = v;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const double o = __shfl_up_sync(0xffffffffu, inc, off);
    if (lane >= off) inc += o;
  }
  __syncthreads();
  if (lane == 31) part[warp] = inc;
  __syncthreads();
  double before = 0.0, all = 0.0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w == warp) before = all;
    all += part[w];
  }
  *total = all;
  return before + inc - v;
}

template <bool LARGEST_FIRST, class U>
__device__ __forceinline__ bool precedes(U a, U b) {
  return LARGEST_FIRST ? a > b : a < b;
}
// A value of each lane, in order.
template <bool LARGEST_FIRST, class U>
__device__ __forceinline__ U sort_warp(U v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1) {
      const U o = __shfl_xor_sync(0xffffffffu, v, j);
      const bool early = ((lane & j) == 0) == ((lane & k) == 0);
      if (precedes<LARGEST_FIRST>(o, v) == early) v = o;
    }
  return v;
}
// V values a thread (of place tid + i * kThreads), n of them, a power of two from 32 on; they lie in order in
// the returned half of buf (twice n).  Warps sort 32 each; of two sorted runs, a value's place in both is its place in
// its own and how many of the other's precede it.
template <bool LARGEST_FIRST, int V, class U>
__device__ __forceinline__ U* sort_threads(U (&v)[V], int n, U* buf) {
  const int tid = threadIdx.x;
  int at[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    at[i] = tid + i * kThreads;
    if (at[i] < n) buf[at[i]] = v[i] = sort_warp<LARGEST_FIRST>(v[i]);
  }
  __syncthreads();
  U *from = buf, *to = buf + n;
  for (int run = 32; run < n; run <<= 1) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (at[i] >= n) continue;
      const U* other = from + ((at[i] & ~(run - 1)) ^ run);
      const bool right = at[i] & run;  // of equal ones the left run's come first
      int before = 0;
      for (int s = run >> 1; s > 0; s >>= 1) {
        const U o = other[before + s - 1];
        if (precedes<LARGEST_FIRST>(o, v[i]) || (right && o == v[i])) before += s;
      }
      const U o = other[before];
      before += precedes<LARGEST_FIRST>(o, v[i]) || (right && o == v[i]);
      at[i] = (at[i] & ~(2 * run - 1)) + (at[i] & (run - 1)) + before;
      to[at[i]] = v[i];
    }
    __syncthreads();
    U* t = from;
    from = to, to = t;
  }
  return from;
}

template <bool RANKS>
constexpr int kHead = (sizeof(Shared) + (RANKS ? sizeof(Ranked) : 0) + 15) / 16 * 16;

// RANKS: some row may have top-k or top-p.
template <class T, bool RANKS>
__global__ void __launch_bounds__(kThreads, 2) sample_tokens_kernel(SampleParams p, int cluster, int slice, int sorted_rows) {
  extern __shared__ __align__(16) uint8_t dynamic[];
  Shared& sh = *reinterpret_cast<Shared*>(dynamic);
  Ranked& rs = *reinterpret_cast<Ranked*>(dynamic + sizeof(Shared));
  T* mine = reinterpret_cast<T*>(dynamic + kHead<RANKS>);
  constexpr int kVec = 16 / sizeof(T);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = blockIdx.x % cluster, warps = cluster * kWarps;
  long long row = blockIdx.x / cluster;
  const int first = rank * slice, n = max(0, min(slice, p.vocab - first));
  for (int i = tid; i < kParts; i += kThreads) sh.table[i] = exp2((double)i / kParts);
  if (tid == 0) sh.listed = 0, sh.first_equal = 0x7fffffff;
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  after_previous();
  if (RANKS && sorted_rows) {  // the rows that may take long, then the others
    const bool there = tid < p.rows;
    const float heat = there && p.temperature ? p.temperature[tid] : 1.f, top_p = there && p.top_p ? p.top_p[tid] : 1.f;
    const int k = there && p.top_k ? p.top_k[tid] : 0;
    const bool may = (heat > 0.f) & (k > 0 && k < p.vocab ? k > kFew : top_p < 1.f);
    const uint32_t votes = __ballot_sync(0xffffffffu, may);
    if (lane == 0) sh.long_rows[warp] = __popc(votes);
    __syncthreads();
    int before = 0, all = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w == warp) before = all;
      all += sh.long_rows[w];
    }
    before += __popc(votes & ((1u << lane) - 1u));
    if (there && (may ? before : all + tid - before) == row) sh.chosen = tid;
    __syncthreads();
    row = sh.chosen;
  }
  const T* src = static_cast<const T*>(p.logits) + row * p.stride + first;
  const float heat = p.temperature ? p.temperature[row] : 1.f;
  const bool greedy = !(heat > 0.f);
  const int k = !RANKS || greedy || !p.top_k ? 0 : p.top_k[row];
  const float top_p = !RANKS || greedy || !p.top_p ? 1.f : p.top_p[row];
  const float min_p = greedy || !p.min_p ? 0.f : p.min_p[row];
  const float u = p.random[row];

  // The row into shared memory: NaN as -inf, -0 as 0; its largest.
  float most = kNone;
  auto clean = [](float v) { return fmaxf(v + 0.f, kNone); };
  int begin = 0;
  const bool even = reinterpret_cast<uintptr_t>(src) % 16 == 0;  // of all of the row's CTAs: slices are whole vectors
  if (even) {
    constexpr int kFlight = 4;
    const int vecs = n / kVec;
    for (int i0 = 0; i0 < vecs; i0 += kFlight * kThreads) {
      uint4 raw[kFlight];
#pragma unroll
      for (int f = 0; f < kFlight; ++f) {
        const int i = i0 + f * kThreads + tid;
        if (i < vecs) raw[f] = reinterpret_cast<const uint4*>(src)[i];
      }
#pragma unroll
      for (int f = 0; f < kFlight; ++f) {
        const int i = i0 + f * kThreads + tid;
        if (i >= vecs) break;
        T* e = reinterpret_cast<T*>(&raw[f]);
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
          const float v = clean(to_f32(e[j]));
          most = fmaxf(most, v);
          e[j] = from_f32<T>(v);
        }
        reinterpret_cast<uint4*>(mine)[i] = raw[f];
      }
    }
    begin = vecs * kVec;
  }
  for (int i = begin + tid; i < n; i += kThreads) {
    const float v = clean(to_f32(src[i]));
    most = fmaxf(most, v);
    mine[i] = from_f32<T>(v);
  }
  // what lies behind, up to a whole vector
  const int padded = (n + kVec - 1) / kVec * kVec;
  if (tid < padded - n) mine[n + tid] = from_f32<T>(kNone);

  __syncwarp();
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // all CTAs run: they may be written to
  // For a list of the row's largest: each warp's each-th largest of its threads', which half of the warps reach at the
  // least.  Few top-k, or, of top-p alone, as many as mostly do.
  const bool by_k = k > 0 && k < p.vocab, by_p = top_p < 1.f;
  const int reach = by_k ? k : by_p ? kReach : 0;
  bool quick = RANKS && reach > 0 && reach <= min(kFew, kWarps / 2 * 32 * cluster);
  const int each = (reach + warps / 2 - 1) / (warps / 2);
  float s = kNone;
  if (quick) {
    s = sort_warp<true>(most);
    if (lane == each - 1)
      for (int r = 0; r < cluster; ++r) *of_rank(&sh.all_level[rank * kWarps + warp], r) = s;
  }
#pragma unroll
  for (int off = 16; off; off >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, off));
  // Of top-p alone, whether that list is likely to do, by the weights of the warp's largest and of a sample of the others, a
  // vector of each thread's: a flat row is spared the pass that would show that it does not.  (All CTAs have to come to one
  // answer, or their barriers part: it goes by what they share, and a slice without a vector has an empty sample.)
  const bool guess = quick && !by_k && even && !(min_p > 0.f);
  const float per_unit = 1.44269504f / heat;
  if (guess) {
    const float level = __shfl_sync(0xffffffffu, s, each - 1);
    float few = lane < each ? exp2f((s - most) * per_unit) : 0.f, sample = 0.f;
    const int own = (n / kVec - tid + kThreads - 1) / kThreads;
    if (own > 0) {
      const uint4 raw = reinterpret_cast<const uint4*>(mine)[tid + warp % own * kThreads];
      const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int j = 0; j < kVec; ++j) sample += to_f32(e[j]) < level ? exp2f((to_f32(e[j]) - most) * per_unit) : 0.f;
      sample *= (float)own;
    }
#pragma unroll
    for (int off = 16; off; off >>= 1) {
      few += __shfl_xor_sync(0xffffffffu, few, off);
      sample += __shfl_xor_sync(0xffffffffu, sample, off);
    }
    if (lane < cluster) {
      *of_rank(&sh.all_few[rank * kWarps + warp], lane) = few;
      *of_rank(&sh.all_sample[rank * kWarps + warp], lane) = sample;
    }
  }
  if (lane < cluster) *of_rank(&sh.all_most[rank * kWarps + warp], lane) = most;
  cluster_sync();
  most = kNone;
  for (int i = lane; i < warps; i += 32) most = fmaxf(most, sh.all_most[i]);
#pragma unroll
  for (int off = 16; off; off >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, off));
  if (guess) {
    float few = 0.f, sample = 0.f;
    for (int i = lane; i < warps; i += 32) {
      const float scale = sh.all_most[i] == kNone ? 0.f : exp2f((sh.all_most[i] - most) * per_unit);
      few += scale > 0.f ? scale * sh.all_few[i] : 0.f;
      sample += scale > 0.f ? scale * sh.all_sample[i] : 0.f;
    }
#pragma unroll
    for (int off = 16; off; off >>= 1) {
      few += __shfl_xor_sync(0xffffffffu, few, off);
      sample += __shfl_xor_sync(0xffffffffu, sample, off);
    }
    quick = !(1.1f * few < top_p * (few + sample));
  }
  if (most == kNone) {
    if (rank == 0 && tid == 0) {
      p.tokens[row] = -1;
      if (p.kept) p.kept[row] = 0;
    }
    return;
  }
  // Vectors of the CTA's slice, by threads: f(index in the slice, values), or of each f(index, value).
  auto for_vectors = [&](int from, int to, int start, int step, auto f) {
    for (int i = from / kVec + start; i < (to + kVec - 1) / kVec; i += step) {
      const uint4 raw = reinterpret_cast<const uint4*>(mine)[i];
      const T* e = reinterpret_cast<const T*>(&raw);
      float l[kVec];
#pragma unroll
      for (int j = 0; j < kVec; ++j) l[j] = to_f32(e[j]);
      f(i * kVec, l);
    }
  };
  auto for_fours = [&](int from, int to, int start, int step, auto f) {
    for_vectors(from, to, start, step, [&](int i, const float(&l)[kVec]) {
#pragma unroll
      for (int j = 0; j < kVec; j += 4) {
        const float four[4] = {l[j], l[j + 1], l[j + 2], l[j + 3]};
        f(i + j, four);
      }
    });
  };
  auto for_all = [&](int from, int to, int start, int step, auto f) {
    for_vectors(from, to, start, step, [&](int i, const float(&l)[kVec]) {
#pragma unroll
      for (int j = 0; j < kVec; ++j) f(i + j, l[j]);
    });
  };

  if (greedy) {
    for_all(0, n, tid, kThreads, [&](int i, float l) {
      if (l == most) atomicMin(&sh.first_equal, i);
    });
    __syncthreads();
    if (tid < cluster) *of_rank(&sh.all_listed[rank], tid) = sh.first_equal;
    cluster_sync();
    if (rank == 0 && tid == 0) {
      int r = 0;
      while (sh.all_listed[r] == 0x7fffffff) ++r;
      p.tokens[row] = r * slice + sh.all_listed[r];
      if (p.kept) p.kept[row] = 1;
    }
    return;
  }

  const bool endless = most == INFINITY;
  // 512 log2 of a weight, from the exact difference.  Where the largest is infinite only its equals are there, at 0.
  const double slope = endless ? 0.0 : kParts * 1.4426950408889634 / (double)heat, top = endless ? kHuge : most;
  auto level_of = [&](float l) -> double { return ((double)l - top) * slope; };  // of a finite l
  // The weight: 2^(y/512) = 2^a 2^(b/512) e^z with whole a and b and |z| <= ln 2 / 1024, for which
  // 1 + z + z^2/2 + z^3/6 is within 9e-15.
  auto weight_at = [&](double y, int& whole) -> double {
    const double shifted = y + kRound;
    whole = __double2loint(shifted);
    const double r = y - (shifted - kRound);
    constexpr double c = 0.6931471805599453 / kParts;
    const double z = fma(r, fma(r, c * c * c / 6, c * c / 2), c);
    const double t = sh.table[whole & (kParts - 1)];
    const double w = fma(t, z * r, t);
    return __hiloint2double(__double2hiint(w) + ((whole & -kParts) << 11), __double2loint(w));
  };
  static_assert(kParts == 512, "");
  // Below it weights, of less than 2^-999.7, count as 0; rounded so that none of less than 2^-1000 is above it.
  const float least_level = endless ? INFINITY : fmaxf(__fsub_ru(most, __fmul_rd(693.f, heat)), -kHuge);
  auto bounded = [&](float l) { return fminf(fmaxf(l, least_level), kHuge); };
  auto weight = [&](float l) -> double {
    int whole;
    const double w = weight_at(level_of(bounded(l)), whole);
    return l >= least_level ? w : 0.0;
  };
  // 64ths of an octave below the largest, in f32: in the order of the values, which is all that is asked of it.  The last
  // bin has whatever is smaller.
  const float per_bin = endless ? 0.f : fmaxf(-64.f * 1.44269504f / heat, -kHuge);
  auto place_of = [&](float l) -> float { return fminf(fmaxf(l - most, -kHuge) * per_bin, kBins - 1.f); };
  auto bin_of = [&](float l) -> int { return (int)place_of(l); };
  // A power of two: units of weight 1 that give the largest weight of a bin, of 2^(-bin / 64), up to 2^bits.  (Those of weight
  // 1 itself would leave few to a weight of 2^-39, of which a vocabulary may hold the goal.  The last bin's are those of its
  // upper end, 2^-32: a weight that is too small for them is too small for a sum of f64 that the row's largest is in.)
  auto units_of_one = [](int bits, int bin) -> double { return __hiloint2double((1023 + bits + bin / 64) << 20, 0); };
  auto units = [&](double w, double one) -> unsigned long long {  // to the nearest
    return (unsigned long long)__double_as_longlong(fma(w, one, kWhole)) & ((1ull << 52) - 1);
  };
  auto units_up = [](double v) -> unsigned long long {  // the least whole number that is not below v, 1 at the least
    const unsigned long long whole = v > 1.0 ? (unsigned long long)v : 1;
    return whole + ((double)whole < v);
  };
  auto entry = [&](float l, int i) -> unsigned long long {
    return (unsigned long long)key_of(from_f32<T>(l)) << 32 | (0xffffffffu - (uint32_t)(first + i));
  };
  auto value_of = [&](uint32_t key) -> float {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
    } else {
      const unsigned short b = (unsigned short)(key & 0x8000u ? key & 0x7fffu : ~key);
      T v;
      memcpy(&v, &b, 2);
      return to_f32(v);
    }
  };
  // Those of all CTAs' lists, one after the other, of place tid + i * kThreads; 0 behind the last.
  auto gather_lists = [&](unsigned long long (&v)[kPer]) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      int at = tid + i * kThreads, r = 0;
      while (r < cluster && at >= sh.all_listed[r]) at -= sh.all_listed[r++];
      v[i] = r < cluster ? of_rank(rs.list, r)[at] : 0;
    }
  };
  auto list = [&](float l, int i) {
    const int at = atomicAdd(&sh.listed, 1);
    if (at < kList) rs.list[at] = entry(l, i);
  };
  const double least = min_p > 0.f ? (double)fminf(min_p, 1.f) : 0.0;
  const double goal_share = u > 0.f ? (double)fminf(u, 1.f) : 0.0;

  if (quick) {
    // the least of the groups' medians: half of each group's warps reach it
    const int groups = (warps + 31) / 32;
    if (warp < groups) {
      const float s = sort_warp<true>(lane < warps ? sh.all_level[warp * 32 + lane] : kNone);
      if (lane == min(32, warps) / 2 - 1) sh.level[warp] = s;
    }
    __syncthreads();
    float level = sh.level[0];
    for (int g = 1; g < groups; ++g) level = fminf(level, sh.level[g]);
    const float bar = fmaxf(level, -kHuge);
    double mass = 0.0, head = 0.0;  // (top-p alone) of all, and of those listed
    if (by_k) {
      for_all(0, n, tid, kThreads, [&](int i, float l) {
        if (l >= bar) list(l, i);
      });
    } else {
      for_fours(0, n, tid, kThreads, [&](int i, const float(&l)[4]) {
        double w[4];
        int whole;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          w[j] = weight_at(level_of(bounded(l[j])), whole);
          w[j] = l[j] >= least_level ? w[j] : 0.0;
        }
        mass += (w[0] + w[1]) + (w[2] + w[3]);
        if (fmaxf(fmaxf(l[0], l[1]), fmaxf(l[2], l[3])) < bar) return;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (l[j] >= bar) {
            list(l[j], i + j);
            head += w[j];
          }
      });
#pragma unroll
      for (int off = 16; off; off >>= 1) {
        mass += __shfl_xor_sync(0xffffffffu, mass, off);
        head += __shfl_xor_sync(0xffffffffu, head, off);
      }
      if (lane < cluster) {
        *of_rank(&sh.all_sum[rank * kWarps + warp], lane) = mass;
        *of_rank(&sh.all_head[rank * kWarps + warp], lane) = head;
      }
    }
    __syncthreads();
    if (tid < cluster) *of_rank(&sh.all_listed[rank], tid) = sh.listed;
    cluster_sync();
    int count = 0;
    bool fits = true;
    for (int r = 0; r < cluster; ++r) count += sh.all_listed[r], fits &= sh.all_listed[r] <= kList;
    fits = fits && count <= (by_k ? kList : kThreads);
    if (!by_k) {  // the list reaches the sum that is wanted, or min_p ends within it, or it holds all
      mass = head = 0.0;
      for (int i = lane; i < warps; i += 32) mass += sh.all_sum[i], head += sh.all_head[i];
#pragma unroll
      for (int off = 16; off; off >>= 1) {
        mass += __shfl_xor_sync(0xffffffffu, mass, off);
        head += __shfl_xor_sync(0xffffffffu, head, off);
      }
      fits = fits && (head >= (double)top_p * mass || weight(bar) < least || bar == -kHuge);
    }
    if (fits) {
      unsigned long long v[kPer] = {};
      if (rank == 0) gather_lists(v);
      cluster_sync();  // no CTA reads another's after this
      if (rank != 0) return;
      int size = 32;
      while (size < count) size <<= 1;
      const unsigned long long* sorted = sort_threads<true, kPer>(v, size, &rs.sorted[0][0]);
      // thread t: the token of rank t
      const bool ranked = tid < (by_k ? min(k, count) : count);
      const unsigned long long mine_of = ranked ? sorted[tid] : 0;
      const int index = (int)(0xffffffffu - (uint32_t)mine_of);
      const double w = ranked ? weight(value_of((uint32_t)(mine_of >> 32))) : 0.0;
      double total;
      const double before = scan_threads(w, sh.scan, &total);
      bool is = ranked && w >= least && (!endless || w > 0.0);
      if (by_p) is = is && (tid == 0 || before < (double)top_p * (by_k ? total : mass));
      const int kept = __syncthreads_count(is);  // a prefix
      if (tid == 0 && p.kept) p.kept[row] = kept;
      // by index; the ranks lead to the weights
      double* weights = reinterpret_cast<double*>(&rs.sorted[0][0]);
      uint32_t* buf = reinterpret_cast<uint32_t*>(&rs.sorted[1][0]);
      weights[tid] = w;
      size = 32;
      while (size < kept) size <<= 1;
      uint32_t by_index[1] = {is ? (uint32_t)index << 9 | (uint32_t)tid : 0xffffffffu};
      __syncthreads();
      const uint32_t* in_order = sort_threads<false, 1>(by_index, size, buf);
      const uint32_t here = tid < kept ? in_order[tid] : 0;
      const double x = tid < kept ? weights[here & 511u] : 0.0;
      const double at = scan_threads(x, sh.scan, &total);
      const double goal = goal_share * total;
      // the first whose end passes the goal, or the last with a weight
      if (tid == 0) sh.first_equal = 0x7fffffff, sh.listed = 0;
      __syncthreads();
      if (x > 0.0) {
        atomicMax(&sh.listed, tid);
        if (at + x > goal) atomicMin(&sh.first_equal, tid);
      }
      __syncthreads();
      if (tid == min(sh.first_equal, sh.listed)) p.tokens[row] = (int)(here >> 9);
      return;
    }
    __syncthreads();
  }

  // Warps own runs of the row, so that the runs' sums stand in the order of the tokens.
  const int run = (slice + kWarps * 32 * kVec - 1) / (kWarps * 32 * kVec) * (32 * kVec);
  const int r0 = min(padded, warp * run), r1 = min(padded, r0 + run);
  double sum = 0.0;  // of the weights of what is kept of the warp's run, over the lanes
  int count = 0;
  bool summed = false;
  // Where the kept ones end: a value, and the last index of it.
  float cut_value = endless ? kHuge : kNone;
  int cut_index = -1;
  auto above_cut = [&](int i, float l) { return l > cut_value || (l == cut_value && first + i <= cut_index); };
  // Moves the cut up: of what is kept so far, the first `share` tokens, or those up to that share of their sum.  The
  // latter, which is the last filter by rank, also sums what is kept.
  auto narrow = [&](bool by_mass, double share) {
    for (int i = tid; i < kBins; i += kThreads) rs.sums[i] = 0;
    if (tid == 0) sh.listed = 0;
    if (tid < kWarps) sh.extra[tid] = 0, sh.extra_count[tid] = 0;
    __syncthreads();
    const bool all_there = cut_value == kNone;
    // Sums of weights are in a bin's own unit, within 1e-5: enough to find the bin, nearly always, and a pass with the exact
    // sums follows anyway.
    for_fours(0, n, tid, kThreads, [&](int i, const float(&l)[4]) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (!(all_there ? l[j] > kNone : above_cut(i + j, l[j]))) continue;
        const float place = place_of(l[j]);
        const int bin = (int)place;
        if (!by_mass)
          atomicAdd(&rs.sums[bin], 1u);
        else if (bin < kBins - 1)
          atomicAdd(&rs.sums[bin], (uint32_t)fmaf(place - (float)bin, -kBinUnit * 0.01077f, kBinUnit));
      }
    });
    cluster_sync();
    // each CTA sums some of the bins over all, in the place of its own, which no other reads before that
    const int per = kBins / cluster;
    for (int bin = rank * per + tid; bin < (rank + 1) * per; bin += kThreads) {
      unsigned long long m = 0;
      for (int r = 0; r < cluster; ++r) m += of_rank(rs.sums, r)[bin];
      rs.sums[bin] = by_mass ? __float_as_uint((float)m * exp2f(bin * (-1.f / 64.f))) : (uint32_t)m;
    }
    cluster_sync();
    constexpr int kEach = kBins / kThreads;
    unsigned long long m[kEach], mass = 0;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int b = tid * kEach + j;
      const uint32_t v = of_rank(rs.sums, b / per)[b];
      mass += m[j] = by_mass ? (unsigned long long)(__uint_as_float(v) * kBinUnit) : v;
    }
    unsigned long long inc = mass;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const unsigned long long o = __shfl_up_sync(0xffffffffu, inc, off);
      if (lane >= off) inc += o;
    }
    if (lane == 31) sh.scan_mass[warp] = inc;
    __syncthreads();
    unsigned long long at = inc - mass, all = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) at += sh.scan_mass[w];
      all += sh.scan_mass[w];
    }
    const double about = by_mass ? share * (double)all : share;
    unsigned long long wanted = (unsigned long long)about;
    wanted = max(1ull, min(all, wanted + ((double)wanted < about)));
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      if (at < wanted && wanted <= at + m[j]) sh.bin = (uint32_t)(tid * kEach + j), sh.above_mass = at;
      at += m[j];
    }
    __syncthreads();
    int bin = (int)sh.bin;
    unsigned long long above = sh.above_mass;
    auto in_bin = [&](int i, float l) { return l > kNone && bin_of(l) == bin && above_cut(i, l); };
    if (by_mass) {
      // What is above the bin is kept, what is in it is listed.  Where the exact sums say that the goal is in another bin, that
      // one, in growing steps until they have it between them.
      int low = 0, high = kBins - 1;
      for (int step = 1;; step *= 2) {
        double mass = 0.0, head = 0.0;
        sum = 0.0, count = 0;
        for_fours(r0, r1, lane, 32, [&](int i, const float(&l)[4]) {
          double w[4];
          int whole;
#pragma unroll
          for (int j = 0; j < 4; ++j) w[j] = weight_at(level_of(bounded(l[j])), whole);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int b = bin_of(l[j]);
            const bool there = l[j] >= least_level && (all_there || above_cut(i + j, l[j]));
            if (there && b == bin) {
              list(l[j], i + j);
              head += w[j];
            }
            w[j] = there ? w[j] : 0.0;
            mass += w[j];
            count += there && b < bin;
            sum += there && b < bin ? w[j] : 0.0;
          }
        });
        double above = sum;
#pragma unroll
        for (int off = 16; off; off >>= 1) {
          mass += __shfl_xor_sync(0xffffffffu, mass, off);
          head += __shfl_xor_sync(0xffffffffu, head, off);
          above += __shfl_xor_sync(0xffffffffu, above, off);
        }
        if (lane < cluster) {
          *of_rank(&sh.all_mass[rank * kWarps + warp], lane) = mass;
          *of_rank(&sh.all_head[rank * kWarps + warp], lane) = head;
          *of_rank(&sh.all_sum[rank * kWarps + warp], lane) = above;
        }
        __syncthreads();
        if (tid < cluster) *of_rank(&sh.all_listed[rank], tid) = sh.listed;
        cluster_sync();
        mass = head = above = 0.0;
        for (int i = lane; i < warps; i += 32) mass += sh.all_mass[i], head += sh.all_head[i], above += sh.all_sum[i];
#pragma unroll
        for (int off = 16; off; off >>= 1) {
          mass += __shfl_xor_sync(0xffffffffu, mass, off);
          head += __shfl_xor_sync(0xffffffffu, head, off);
          above += __shfl_xor_sync(0xffffffffu, above, off);
        }
        const double goal = share * mass;
        const bool before = above >= goal && bin > 0, behind = !before && above + head < goal;
        if (before) high = bin - 1;
        if (behind) low = bin + 1;
        if (!(before || behind) || step == 0 || (behind && low > high)) {
          if (tid == 0) sh.rest = goal - above, sh.rest_bin = bin;
          break;
        }
        if (low > high) {  // on a border, where the sums of its sides, added up in different ways, differ: what lies before it
          bin = high;
          step = 0;
        } else {
          bin = before ? max(low, bin - step) : min(high, bin + step);
          if (low > 0 && high < kBins - 1) bin = (low + high) / 2;
        }
        cluster_sync();  // all have read what the next pass writes
        if (tid == 0) sh.listed = 0;
        __syncthreads();
      }
      above = 0;
    } else {
      for_all(0, n, tid, kThreads, [&](int i, float l) {
        if (in_bin(i, l)) list(l, i);
      });
      __syncthreads();
      if (tid < cluster) *of_rank(&sh.all_listed[rank], tid) = sh.listed;
      cluster_sync();
    }
    int entries = 0;
    bool fits = true;
    for (int r = 0; r < cluster; ++r) entries += sh.all_listed[r], fits &= sh.all_listed[r] <= kList;
    fits = fits && entries <= kList;
    if (fits) {
      if (rank == 0) {
        unsigned long long v[kPer];
        gather_lists(v);
        int size = 32;
        while (size < entries) size <<= 1;
        // thread t: ranks from kPer t on
        const unsigned long long* sorted = sort_threads<true, kPer>(v, size, &rs.sorted[0][0]);
        if (tid == 0) sh.first_equal = entries - 1;
        __syncthreads();
        const double one = units_of_one(kListBits, sh.rest_bin);
        if (by_mass) wanted = units_up(sh.rest * one);
        unsigned long long own[kPer], sum = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          v[i] = kPer * tid + i < entries ? sorted[kPer * tid + i] : 0;
          own[i] = kPer * tid + i >= entries ? 0 : by_mass ? units(weight(value_of((uint32_t)(v[i] >> 32))), one) : 1;
          sum += own[i];
        }
        inc = sum;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
          const unsigned long long o = __shfl_up_sync(0xffffffffu, inc, off);
          if (lane >= off) inc += o;
        }
        if (lane == 31) sh.scan_mass[warp] = inc;
        __syncthreads();
        unsigned long long passed = above + inc - sum;
        for (int w = 0; w < warp; ++w) passed += sh.scan_mass[w];
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          passed += own[i];
          if (kPer * tid + i < entries && passed >= wanted) atomicMin(&sh.first_equal, kPer * tid + i);
        }
        __syncthreads();
        if (tid < cluster) {
          const unsigned long long last = entries > 0 ? sorted[sh.first_equal] : entry(most, 0x7fffffff - first);
          *of_rank(&sh.cut_key, tid) = (uint32_t)(last >> 32);
          *of_rank(&sh.cut_index, tid) = (int)(0xffffffffu - (uint32_t)last);
        }
      }
      cluster_sync();
      cut_value = value_of(sh.cut_key), cut_index = sh.cut_index;
      if (by_mass && least == 0.0) {
        // the kept of the bin, in whole units: listed in any order, their sums are the same
        const double one = units_of_one(kListBits, sh.rest_bin);
        for (int i = tid; i < sh.listed; i += kThreads) {
          const unsigned long long v = rs.list[i];
          const int at = (int)(0xffffffffu - (uint32_t)v) - first;
          const float l = value_of((uint32_t)(v >> 32));
          if (above_cut(at, l)) {
            atomicAdd(&sh.extra[at / run], units(weight(l), one));
            atomicAdd(&sh.extra_count[at / run], 1);
          }
        }
        __syncthreads();
        if (lane == 0) sum += (double)sh.extra[warp] / one, count += sh.extra_count[warp];
        summed = true;
      }
      if (!summed) sum = 0.0, count = 0;
      return;
    }
    // More of nearly one value than a list holds: by descending digits of their keys.
    sum = 0.0, count = 0;
    uint32_t known = 0, key_so_far = 0;
    unsigned long long before = above, equal = 0, equal_mass = 0;
    for (int high = kKeyBits<T>; high > 0;) {
      const int digit = min(11, high), shift = high - digit;
      for (int i = tid; i < kBins; i += kThreads) rs.digits.count[i] = 0, rs.digits.mass[i] = 0;
      __syncthreads();
      for_all(0, n, tid, kThreads, [&](int i, float l) {
        const uint32_t key = key_of(from_f32<T>(l));
        if ((key & known) == key_so_far && in_bin(i, l)) {
          const uint32_t b = key >> shift & ((1u << digit) - 1u);
          atomicAdd(&rs.digits.count[b], 1u);
          if (by_mass) atomicAdd(&rs.digits.mass[b], units(weight(l), units_of_one(kRowBits, sh.rest_bin)));
        }
      });
      cluster_sync();
      // thread t sums four bins over the CTAs, from the top down
      uint32_t c[kEach];
      mass = 0;
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        const int b = kBins - 1 - (tid * kEach + j);
        c[j] = 0, m[j] = 0;
        for (int r = 0; r < cluster; ++r) c[j] += of_rank(rs.digits.count, r)[b], m[j] += of_rank(rs.digits.mass, r)[b];
        if (!by_mass) m[j] = c[j];
        mass += m[j];
      }
      inc = mass;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const unsigned long long o = __shfl_up_sync(0xffffffffu, inc, off);
        if (lane >= off) inc += o;
      }
      if (lane == 31) sh.scan_mass[warp] = inc;
      __syncthreads();
      at = before + inc - mass, all = before;
      for (int w = 0; w < kWarps; ++w) {
        if (w < warp) at += sh.scan_mass[w];
        all += sh.scan_mass[w];
      }
      if (by_mass && known == 0) wanted = min(units_up(sh.rest * units_of_one(kRowBits, sh.rest_bin)), all);  // (rounded otherwise than the sums of weights)
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        if (at < wanted && wanted <= at + m[j]) {
          sh.bin = kBins - 1 - (tid * kEach + j);
          sh.above_mass = at, sh.bin_mass = m[j], sh.bin_count = c[j];
        }
        at += m[j];
      }
      cluster_sync();
      before = sh.above_mass, equal = sh.bin_count, equal_mass = sh.bin_mass;
      key_so_far |= sh.bin << shift;
      known |= ((1u << digit) - 1u) << shift;
      high = shift;
      __syncthreads();
    }
    // Of those with that key the first, by index.
    const unsigned long long a_tie = equal_mass / equal, ties = min(equal, (wanted - before + a_tie - 1) / a_tie);
    const float cut = value_of(key_so_far);
    int same = 0;
    for (int i = r0 + lane; i < min(r1, n); i += 32) same += to_f32(mine[i]) == cut && above_cut(i, cut);
    same = __reduce_add_sync(0xffffffffu, same);
    if (lane < cluster) *of_rank(&sh.all_equal[rank * kWarps + warp], lane) = same;
    cluster_sync();
    unsigned long long earlier = 0;
    for (int i = 0; i < rank * kWarps + warp; ++i) earlier += sh.all_equal[i];
    if (earlier < ties && ties <= earlier + same) {
      for (int i0 = r0; i0 < min(r1, n); i0 += 32) {
        const int i = i0 + lane;
        const bool is = i < min(r1, n) && to_f32(mine[i]) == cut && above_cut(i, cut);
        const uint32_t votes = __ballot_sync(0xffffffffu, is);
        if (earlier + __popc(votes) >= ties) {
          if (is && __popc(votes & (0xffffffffu >> (31 - lane))) == (int)(ties - earlier))
            for (int r = 0; r < cluster; ++r) *of_rank(&sh.cut_index, r) = first + i;
          break;
        }
        earlier += __popc(votes);
      }
    }
    cluster_sync();
    cut_value = cut, cut_index = sh.cut_index;
  };
  if (RANKS) {
#pragma unroll 1
    for (int mass = by_k ? 0 : 1; mass <= (by_p ? 1 : 0); ++mass) narrow(mass != 0, mass ? (double)fmaxf(top_p, 0.f) : (double)k);
  }

  // 0 where the token is not kept
  auto kept_weight = [&](int i, float l) -> double {
    const double w = weight(l);
    return above_cut(i, l) && w >= least ? w : 0.0;
  };
  if (!summed) {
    const bool plain = !by_k && !by_p && least == 0.0 && !endless;  // all that are there
    for_fours(r0, r1, lane, 32, [&](int i, const float(&l)[4]) {
      bool is[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) is[j] = plain ? l[j] > kNone : above_cut(i + j, l[j]);
      if (!(is[0] | is[1] | is[2] | is[3])) return;
      double w[4];
      int whole;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        w[j] = weight_at(level_of(bounded(l[j])), whole);
        w[j] = is[j] && l[j] >= least_level ? w[j] : 0.0;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (!plain) {
          is[j] = is[j] && w[j] >= least;
          w[j] = is[j] ? w[j] : 0.0;
        }
        count += is[j];
      }
      sum += (w[0] + w[1]) + (w[2] + w[3]);
    });
  }
#pragma unroll
  for (int off = 16; off; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  count = __reduce_add_sync(0xffffffffu, count);
  if (lane < cluster) {
    *of_rank(&sh.all_sum[rank * kWarps + warp], lane) = sum;
    *of_rank(&sh.all_count[rank * kWarps + warp], lane) = count;
  }
  cluster_sync();  // no CTA reads or writes another's after this
  // The run in which the sum passes the goal; the last with a sum where rounding keeps it from that.
  constexpr int kEachRun = kMaxWarps / 32;
  double sums[kEachRun], mine_sum = 0.0;
  int all = 0;
#pragma unroll
  for (int j = 0; j < kEachRun; ++j) {
    const int i = lane * kEachRun + j;
    sums[j] = i < warps ? sh.all_sum[i] : 0.0;
    mine_sum += sums[j];
    all += i < warps ? sh.all_count[i] : 0;
  }
  double upto = mine_sum;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const double o = __shfl_up_sync(0xffffffffu, upto, off);
    if (lane >= off) upto += o;
  }
  const double goal = goal_share * __shfl_sync(0xffffffffu, upto, 31);
  int owner = -1, last_run = -1;
  double before = upto - mine_sum, last_before = 0.0, owner_before = 0.0;
#pragma unroll
  for (int j = 0; j < kEachRun; ++j) {
    if (sums[j] > 0.0) {
      last_run = lane * kEachRun + j, last_before = before;
      if (owner < 0 && before + sums[j] > goal) owner = last_run, owner_before = before;
    }
    before += sums[j];
  }
  const uint32_t passing = __ballot_sync(0xffffffffu, owner >= 0), any = __ballot_sync(0xffffffffu, last_run >= 0);
  const int from = passing ? __ffs(passing) - 1 : 31 - __clz(any);
  owner = __shfl_sync(0xffffffffu, passing ? owner : last_run, from);
  before = __shfl_sync(0xffffffffu, passing ? owner_before : last_before, from);
  all = __reduce_add_sync(0xffffffffu, all);
  if (rank == 0 && tid == 0 && p.kept) p.kept[row] = all;
  if (owner / kWarps != rank) return;
  // All threads on that run, consecutive tokens each.
  const int w0 = min(n, owner % kWarps * run), w1 = min(n, w0 + run), share = (run + kThreads - 1) / kThreads;
  const int i0 = min(w1, w0 + tid * share), i1 = min(w1, i0 + share);
  double part = 0.0, ignored;
  for (int i = i0; i < i1; ++i) part += kept_weight(i, to_f32(mine[i]));
  if (tid == 0) sh.first_equal = 0x7fffffff, sh.listed = -1;
  const double lo = before + scan_threads(part, sh.scan, &ignored);
  // the first thread whose end passes the goal, or the last with a sum
  if (part > 0.0) {
    atomicMax(&sh.listed, tid);
    if (lo + part > goal) atomicMin(&sh.first_equal, tid);
  }
  __syncthreads();
  if (tid == min(sh.first_equal, sh.listed)) {
    double running = lo;
    int token = -1;
    for (int i = i0; i < i1; ++i) {
      const double w = kept_weight(i, to_f32(mine[i]));
      if (w > 0.0) {
        token = first + i;
        running += w;
        if (running > goal) break;
      }
    }
    p.tokens[row] = token;
  }
}

template <class T, bool RANKS>
cudaError_t launch_sample(const SampleParams& p, int cluster, int sm_count, cudaStream_t st) {
  constexpr int kMaxDevices = 64, kMaxBytes = 227 * 1024;
  static_assert(kSampleMaxVocab / kMaxCluster * (double)kBinUnit < 4294967296.0 && kMostBytes / 2 * (double)kBinUnit < 4294967296.0, "a CTA's bins");
  static_assert(kHead<RANKS> + kSampleMaxVocab / kMaxCluster * (int)sizeof(T) <= kMaxBytes, "");
  static std::atomic<unsigned> asked[kMaxDevices];
  const int slice = ((p.vocab + cluster - 1) / cluster + 7) / 8 * 8, smem = kHead<RANKS> + slice * (int)sizeof(T);
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const unsigned gen = attr_generation(dev) + 1;
  if (dev >= kMaxDevices || asked[dev].load(std::memory_order_acquire) != gen) {
    e = cudaFuncSetAttribute(sample_tokens_kernel<T, RANKS>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxBytes);
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
  // More CTAs than run at once: the last to start should not be those that take longest (the mixture above 55 us as they come;
  // it costs 1 where no row takes long).
  const int sorted_rows = p.rows <= kThreads && (long long)p.rows * cluster > 2 * sm_count;
  return cudaLaunchKernelEx(&cfg, sample_tokens_kernel<T, RANKS>, p, cluster, slice, sorted_rows);
}

template <class T>
cudaError_t launch_sample(const SampleParams& p, int sm_count, cudaStream_t st) {
  const bool ranks = p.top_k || p.top_p;
  const int head = ranks ? kHead<true> : kHead<false>;
  // CTAs of a row: as its size needs them where two share a SM; more, without ranks, until there is about one a SM; with
  // them until there are two, and with both top-k and top-p, where rows that go without top-k may take long, until there
  // are four, of which two run at once.  us with 2, 4, 8: 64 x 128256 bf16, plain 23, 22.5, 29; top-k of all rows -, 20.6, 31.9; flat
  // rows with top-p alone 101, 60, 75; a mixture 72, 56, 44, though 20, 19.5, 31 where all its rows have top-k.  With 1, 2, 4:
  // 256 x 32000 f32, all filters 36, 33, 46, plain 30, 27, 36.
  int cluster = 1;
  while (cluster < kMaxCluster &&
         ((ranks ? (long long)p.rows * cluster * 2 <= (p.top_k && p.top_p ? 4 : 2) * sm_count : (long long)p.rows * cluster * 10 < 8 * sm_count) ||
          head + ((p.vocab + cluster - 1) / cluster + 8) * (int)sizeof(T) > kMostBytes))
    cluster *= 2;
  return ranks ? launch_sample<T, true>(p, cluster, sm_count, st) : launch_sample<T, false>(p, cluster, sm_count, st);
}

}  // namespace

cudaError_t launch_sample_tokens(const SampleParams& p, int dtype, int sm_count, cudaStream_t st) {
  if (dtype == kTypeF32) return launch_sample<float>(p, sm_count, st);
  return dtype == kTypeBF16 ? launch_sample<__nv_bfloat16>(p, sm_count, st) : launch_sample<__half>(p, sm_count, st);
}

}  // namespace tk
