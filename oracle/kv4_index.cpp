// The index arithmetic of the 4-bit cache's operators (tk_kv4.h), compiled for the CPU tests.
#include "../tiny-kernel_b200/csrc/tk_kv4.h"

using namespace tk;

extern "C" {

long long kv4_index_slot_row(int num_blocks, int kv_heads, int shift, int slot, int head) {
  Kv4View c{};
  c.num_blocks = num_blocks;
  c.kv_heads = kv_heads;
  c.shift = shift;
  return kv4_slot_row(c, slot, head);
}

long long kv4_index_row(int num_blocks, int kv_heads, int shift, int block, int head, int off) {
  Kv4View c{};
  c.num_blocks = num_blocks;
  c.kv_heads = kv_heads;
  c.shift = shift;
  return kv4_row(c, block, head, off);
}

int kv4_index_wanted(int ctx, int q) { return slots_wanted(ctx, q); }

// out: ctx, q, have, need
void kv4_index_request(int ctx, int q, long long start, int shift, int max_blocks, int max_tokens, int* out) {
  const SlotsRequest r = slots_request(ctx, q, start, shift, max_blocks, max_tokens);
  out[0] = r.ctx;
  out[1] = r.q;
  out[2] = r.have;
  out[3] = r.need;
}

int kv4_index_tokens_in(int ctx, int q, int j, int shift) {
  const SlotsRequest r{ctx, q, 0, 0};
  return slots_tokens_in(r, j, shift);
}

long long kv4_index_prompt_work(int tiles, int per, int cost, int last, int kv) {
  return prompt_work(prompt_tiles(tiles, per, cost, last, kv));
}
int kv4_index_prompt_steps(int tiles, int per, int cost, int last, int kv, int tile) {
  return prompt_steps(prompt_tiles(tiles, per, cost, last, kv), tile);
}
int kv4_index_prompt_find(int tiles, int per, int cost, int last, int kv, long long x, int* at) {
  return prompt_find(prompt_tiles(tiles, per, cost, last, kv), x, at);
}

int kv4_index_new_block(const int* list, int begin, int end, long long a, int num_blocks) {
  return slots_new_block(list, begin, end, a, num_blocks);
}
}
