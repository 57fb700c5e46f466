// What the paged-attention kernels share: the plan's records, the problem's
// description, and the arithmetic of one score.
//
// For query row i of a request (position p_i = kv_len - q_len + i), head h,
// and key j of its paged sequence,
//   s_ij = cap * tanh(scale * q_i . k_j / cap)      (cap > 0, else scale * q_i . k_j)
//          - slope_h * |p_i - j|                    (with slopes)
//   o_i  = sum_j e^(s_ij - m_i) v_j / sum_j e^(s_ij - m_i),   j in lo_i <= j < hi_i
// Every mask but a tree's is an interval [lo_i, hi_i) of keys: causal order,
// a bidirectional prefix, a sliding window and a packed document each move one
// of its ends.  A tree of drafted tokens adds single keys past hi_i, one bit
// each.  A row that sees no key is zero.
#pragma once

#include "fp8.cuh"

namespace pace {
namespace attn {

// Per query token, from the plan: visible keys [lo, hi), the request's first
// entry in kv_indices, and the token's position (with a tree, the sequence's
// length: its drafted keys are hi .. pos - 1).
struct TokenInfo {
  int lo, hi, page_base, pos;
};

// A piece of work: `ntok` query tokens (all their heads of one kv head) over
// keys [kv_begin, kv_end).  splits > 1: it is number `split` of that many
// pieces of the same rows, which leave partial results in slots `slot`,
// slot + 1, ... and count their arrivals in counter `tile`.
struct Item {
  int tok0, ntok, kv_begin, kv_end;
  int page_base, tile, slot, split;
  int splits, pad0, pad1, pad2;
};
static_assert(sizeof(Item) == 48 && sizeof(TokenInfo) == 16, "plan records are int32 words");

constexpr float kLog2e = 1.4426950408889634f;

struct Problem {
  const void* query;  // [total_q, heads, head_dim], tokens q_stride apart
  void* out;
  const void* cache;           // 16-bit or fp32 pages, or e4m3 codes
  const uint8_t* exponents;    // codes' exponents, or null
  const int32_t* kv_indices;
  const TokenInfo* tokens;
  const float* slopes;         // per query head, or null
  const uint64_t* tree_mask;   // [total_q, tree_words], or null
  float* lse;                  // [total_q, heads] natural log, or null
  int64_t q_stride, out_stride;
  int64_t total_q;
  int heads, kv_heads, head_dim, page_size, tree_words;
  float scale;  // of q . k
  float cap;    // 0: none
};

// One score in natural units.
__device__ __forceinline__ float score(float dot, float scale, float cap, float slope, int distance) {
  float s = dot * scale;
  if (cap > 0.f) s = cap * tanhf(s / cap);
  return s - slope * (float)distance;
}

// Whether drafted token `node` (0 .. 64 * words - 1) is visible.
__device__ __forceinline__ bool tree_bit(const uint64_t* row, int node) {
  return (row[node >> 6] >> (node & 63)) & 1u;
}

}  // namespace attn
}  // namespace pace
