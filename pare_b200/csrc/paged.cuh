// Shared by the kernels of the paged 8-bit KV cache (paged_cache.cu, paged_attn.cu): the layout of a step's tables.
#pragma once

#include "common.cuh"

namespace pare {
namespace paged {

constexpr int kMaxRequests = 4096;
constexpr int kMaxQueryTokens = 4096;      // tokens of a step that attention is planned for
constexpr int kMaxTokens = 1 << 22;
constexpr int kUnit = 16;                  // tokens per unit of attention work
constexpr int kPacks = 4;                  // attention tiles of 1, 2, 4, 8 tokens of a request: a table of units for each
constexpr int kItemInts = 8;               // request, block id, first row, offset in the block, tokens, block index, length before, length after

// Whether tokens of a request share tiles: where there are more rows than requests, some request has several new tokens.  (8 requests x
// 8 tokens over 2000, 16 query and KV heads: 191 -> 86 us for two layers.)
__host__ __device__ inline bool packs_tokens(int R, int T) { return T > R; }

inline bool block_size_ok(int bs) { return bs == 16 || bs == 32 || bs == 64; }

// Blocks that T new tokens of at most R requests touch: one per token at most; a request with n tokens touches ceil((n - 1) / bs) + 1.
inline int max_items(int R, int T, int bs) {
  const int64_t a = (int64_t)T / bs + 2ll * (R < T ? R : T);
  return (int)(a < T ? a : T);
}

// A step: one buffer of 32-bit words, every array on a 16-byte boundary.
struct StepLayout {
  int64_t status, query_start, seq_lens, context_start, token_request, positions, slots, unit_start, unit_stride, info, items, words;
  int n_items;
  bool units;
  __host__ StepLayout(int R, int T, int bs) {
    auto up = [](int64_t w) { return (w + 3) / 4 * 4; };
    n_items = max_items(R, T, bs);
    units = T <= kMaxQueryTokens;
    status = 0;
    query_start = 4;
    seq_lens = query_start + up(R + 1);            // [R] lengths, then the number of free blocks
    context_start = seq_lens + up(R + 1);          // [R + 1] 64-bit
    slots = context_start + up(2 * ((int64_t)R + 1));   // [T] 64-bit
    token_request = slots + up(2 * (int64_t)T);
    positions = token_request + up(T);
    unit_start = positions + up(T);
    unit_stride = up((int64_t)T + 1);
    info = unit_start + (units ? kPacks * unit_stride : 0);     // [T] request, position, length after the step, number in the request's rows
    items = info + (units ? 4 * (int64_t)T : 0);
    words = items + (int64_t)n_items * kItemInts;
  }
};

// What append, dense and attention ask of their layer and step
inline int check(const pare_paged_layer* l, const pare_paged_tables* t) {
  PARE_REQUIRE(l && t && t->step && t->block_table && l->k_codes && l->v_codes && l->k_scale && l->v_scale && l->tail_k && l->tail_v, PARE_ERR_SHAPE);
  PARE_REQUIRE(t->R > 0 && t->R <= kMaxRequests && t->T >= 0 && t->T <= kMaxTokens && t->max_blocks > 0 && t->ld_table >= t->max_blocks, PARE_ERR_SHAPE);
  PARE_REQUIRE(l->num_blocks > 0 && l->H > 0 && l->H <= 65535 && l->R == t->R && l->block_size == t->block_size, PARE_ERR_SHAPE);
  PARE_REQUIRE(l->dtype == PARE_F16 || l->dtype == PARE_BF16, PARE_ERR_DTYPE);
  PARE_REQUIRE(block_size_ok(l->block_size) && (l->D == 64 || l->D == 128), PARE_ERR_UNSUPPORTED);
  PARE_REQUIRE(aligned16(t->step) && aligned16(l->k_codes) && aligned16(l->v_codes) && aligned16(l->tail_k) && aligned16(l->tail_v), PARE_ERR_ALIGN);
  return PARE_OK;
}

}  // namespace paged
}  // namespace pare
