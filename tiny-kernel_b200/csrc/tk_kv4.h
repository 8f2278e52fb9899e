// tk_kv4.h -- the key/value cache held in 4 bits: its index arithmetic and the launchers of the
// operators around it (tk_kv4.cu, tk_kv4_attention.cu).
//
// Everything that turns a device-side value (a slot, a block id, a length) into an address goes
// through the functions here, which refuse what lies outside the cache.  They compile for the host
// too, where the CPU tests run them over good and bad values.
#pragma once
#include <cstddef>
#include <cstdint>

#if defined(__CUDACC__)
#define TK_HD __host__ __device__ __forceinline__
#else
#define TK_HD inline
#endif

namespace tk {

// Element types of activations (TK_F32, TK_F16, TK_BF16 of the ABI).
enum : int { kTypeF32 = 0, kTypeF16 = 1, kTypeBF16 = 2 };

// The cache: codes [block][kv_head][block_size][head_dim / 2] (even dimension in the low nibble)
// and (scale, offset) f16 pairs [block][kv_head][block_size][head_dim / group]; value = code * scale
// + offset.  block_size is a power of two (1 << shift).
struct Kv4View {
  uint8_t* k_codes;
  uint8_t* v_codes;
  uint32_t* k_scales;  // one f16 pair per word: scale in the low half
  uint32_t* v_scales;
  int num_blocks, kv_heads, shift, head_dim, group;
};

// Row (of head_dim values) of token `off` of a block, or -1 for a block outside the cache.  64-bit:
// a cache of 180 GB has more than 2^32 bytes, and more than 2^31 rows at one head dimension of 64.
TK_HD long long kv4_row(const Kv4View& c, int block, int head, int off) {
  if (block < 0 || block >= c.num_blocks) return -1;
  return (((long long)block * c.kv_heads + head) << c.shift) + off;
}

// Row of a slot (block * block_size + token in the block), or -1 for a slot outside the cache.
TK_HD long long kv4_slot_row(const Kv4View& c, int slot, int head) {
  if (slot < 0) return -1;
  return kv4_row(c, slot >> c.shift, head, slot & ((1 << c.shift) - 1));
}

// ---- block tables and slots of a step ------------------------------------------------------------

struct SlotsParams {
  const int* context_lens;  // [batch] tokens in the cache
  const int* query_lens;    // [batch] tokens of this step
  const int* free_blocks;   // ids the step may take: [free_range[0], free_range[1])
  const int* free_range;
  int* block_tables;  // [batch][max_blocks]
  int* kv_lens;       // [batch]
  int* query_start;   // [batch + 1]
  int* positions;     // [max_tokens]
  int* slots;         // [max_tokens]
  int* counts;        // {tokens, blocks taken, tokens without a slot, next free index}
  int batch, max_blocks, shift, num_blocks, max_tokens;
};

// A request within the step: its lengths as they count, and the pages it has and needs.
struct SlotsRequest {
  int ctx, q;      // tokens in the cache, tokens of this step
  int have, need;  // pages in use before and after, at most max_blocks
};

// Tokens that a request asks for: its last position is one that an int holds.
TK_HD int slots_wanted(int ctx, int q) {
  const int top = 0x7fffffff - (ctx > 0 ? ctx : 0);
  return q <= 0 ? 0 : (q < top ? q : top);
}

// start: tokens that the requests before it ask for.  The step's tokens stop at max_tokens.
TK_HD SlotsRequest slots_request(int ctx, int q, long long start, int shift, int max_blocks,
                                 int max_tokens) {
  SlotsRequest r;
  r.ctx = ctx > 0 ? ctx : 0;
  const long long room = max_tokens - start;
  long long n = slots_wanted(ctx, q);
  n = n < room ? n : (room > 0 ? room : 0);
  r.q = (int)n;
  const long long bs1 = (1ll << shift) - 1;
  const long long have = (r.ctx + bs1) >> shift;
  const long long need = n > 0 ? (r.ctx + n + bs1) >> shift : have;
  r.have = (int)(have < max_blocks ? have : max_blocks);
  r.need = (int)(need < max_blocks ? need : max_blocks);
  return r;
}

// Tokens of the request in its page j.
TK_HD int slots_tokens_in(const SlotsRequest& r, int j, int shift) {
  const long long lo = (long long)j << shift, hi = lo + (1ll << shift), kv = (long long)r.ctx + r.q;
  const long long n = (hi < kv ? hi : kv) - (lo > r.ctx ? lo : r.ctx);
  return n > 0 ? (int)n : 0;
}

// The id of the a-th page that the step takes, -1 when the pool is out or the id is none of the
// cache's.  The range starts at 0 at the least; nothing at or past its end is read.
TK_HD int slots_new_block(const int* free_blocks, int begin, int end, long long a, int num_blocks) {
  const long long i = (begin > 0 ? begin : 0) + a;
  if (i >= end) return -1;
  const int id = free_blocks[i];
  return id >= 0 && id < num_blocks ? id : -1;
}

// ---- the work of a prompt ------------------------------------------------------------------------

// Tiles of 128 rows (query token, head of the group) of a sequence against steps of 128 positions: the
// tiles of 128 tokens, `per` of them, count as many steps as the last of those tokens sees, and `cost`.
// So the steps grow by one from each `per` tiles to the next, and their sums have a closed form.
struct PromptTiles {
  int tiles, per, cost;
  int base;  // steps that the token before the first sees; negative where it sees nothing
  int most;  // of the sequence
};
TK_HD PromptTiles prompt_tiles(int tiles, int per, int cost, int last, int kv) {  // last: kv_len less the query tokens
  const int base = last > 0 ? last / 128 + (last % 128 != 0) : last / 128;
  return {tiles, per, cost, base, kv / 128 + (kv % 128 != 0)};
}
TK_HD int prompt_steps(const PromptTiles& t, int tile) {
  const int i = t.base + tile / t.per + 1;
  return t.cost + (i < 0 ? 0 : i < t.most ? i : t.most);
}
// The sum of i up to x, each within 0 .. most.
TK_HD long long prompt_sum(long long x, long long most) {
  return x <= 0 ? 0 : x <= most ? x * (x + 1) / 2 : most * (most + 1) / 2 + (x - most) * most;
}
// Steps of the first n times `per` tiles.
TK_HD long long prompt_before(const PromptTiles& t, int n) {
  return t.per * (prompt_sum((long long)t.base + n, t.most) - prompt_sum(t.base, t.most) + (long long)t.cost * n);
}
TK_HD long long prompt_work(const PromptTiles& t) {
  const int n = t.tiles / t.per, rest = t.tiles - n * t.per;
  return prompt_before(t, n) + (rest ? (long long)rest * prompt_steps(t, n * t.per) : 0);
}
// The tile that step x of all (below prompt_work) lies in, and its place there.
TK_HD int prompt_find(const PromptTiles& t, long long x, int* at) {
  int lo = 0, hi = t.tiles / t.per;
  while (lo < hi) {
    const int mid = lo + (hi - lo + 1) / 2;
    if (prompt_before(t, mid) <= x)
      lo = mid;
    else
      hi = mid - 1;
  }
  const long long rest = x - prompt_before(t, lo);
  const int steps = prompt_steps(t, lo * t.per), i = (int)(rest / steps);
  *at = (int)(rest - (long long)i * steps);
  return lo * t.per + i;
}

}  // namespace tk

#if defined(__CUDACC__)
#include <cuda_runtime.h>

namespace tk {

// tk_kv4.cu
cudaError_t launch_paged_slots(const SlotsParams& p, int sm_count, cudaStream_t st);

struct QkNormRopeParams {
  const void* x[2];        // q, k: rows of heads * head_dim values, in_stride elements apart
  void* out[2];
  const float* weight[2];  // [head_dim] or null: no norm
  long long in_stride[2], out_stride[2];
  int heads[2];
  const float* cos_cache;  // [max_pos][rot_dim / 2]
  const float* sin_cache;
  const int* positions;    // [tokens]
  int tokens, head_dim, rot_dim, max_pos, interleaved;
  float eps;
};
cudaError_t launch_qk_norm_rope(const QkNormRopeParams& p, int dtype, int sm_count, cudaStream_t st);

// k, v: rows of kv_heads * head_dim values, stride elements apart; slots [tokens].
cudaError_t launch_kv4_append(const Kv4View& c, const void* k, const void* v, const int* slots,
                              int tokens, long long k_stride, long long v_stride, int dtype,
                              int sm_count, cudaStream_t st);
cudaError_t launch_kv4_gather(const Kv4View& c, void* k, void* v, const int* slots, int tokens,
                              long long k_stride, long long v_stride, int dtype, int sm_count,
                              cudaStream_t st);

// tk_kv4_attention.cu
struct Kv4AttentionParams {
  Kv4View cache;
  const void* q;  // [tokens] rows of q_heads * head_dim values, q_stride elements apart
  void* o;
  const int* block_tables;  // [batch][max_blocks]
  const int* kv_lens;       // [batch] tokens in the cache, this step's among them
  const int* query_start;   // [batch + 1], null: one query token per sequence
  void* workspace;
  long long q_stride, o_stride;
  int tokens, batch, q_heads, max_blocks;
  float scale;
  double inv_ctas;  // 1 / CTAs, set at the launch
  unsigned* err;    // the device's error word, and how long a wait of a kernel may take
  unsigned long long timeout_ns;
};
size_t kv4_attention_workspace(int head_dim, int sm_count);
cudaError_t launch_kv4_attention(const Kv4AttentionParams& p, int dtype, int sm_count,
                                 cudaStream_t st);

}  // namespace tk
#endif
