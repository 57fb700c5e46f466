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
// slot + 1, ... and count their arrivals in counter `tile`.  mixed: some row
// may not see every key of the piece's rows.  all_begin, all_end: the keys of all
// pieces of these rows.
struct Item {
  int tok0, ntok, kv_begin, kv_end;
  int page_base, tile, slot, split;
  int splits, mixed, all_begin, all_end;
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
  int page_shift;  // log2 of the page size; -1: no power of two
  float scale;  // of q . k
  float cap;    // 0: none
};

// One score in natural units.
__device__ __forceinline__ float score(float dot, float scale, float cap, float slope, int distance) {
  float s = dot * scale;
  if (cap > 0.f) s = cap * tanhf(s / cap);
  return s - slope * (float)distance;
}

// Page and slot of a position, without the division where there need be none.
__device__ __forceinline__ int page_number(const Problem& p, int pos) {
  return p.page_shift >= 0 ? pos >> p.page_shift : pos / p.page_size;
}
__device__ __forceinline__ int page_slot(const Problem& p, int pos) {
  return p.page_shift >= 0 ? pos & (p.page_size - 1) : pos % p.page_size;
}

// Whether drafted token `node` (0 .. 64 * words - 1) is visible.
__device__ __forceinline__ bool tree_bit(const uint64_t* row, int node) {
  return (row[node >> 6] >> (node & 63)) & 1u;
}

template <typename KV>
__device__ __forceinline__ float load_kv(const KV* p, float) {
  return Traits<KV>::to_f(*p);
}
template <>
__device__ __forceinline__ float load_kv<uint8_t>(const uint8_t* p, float factor) {
  float f[4];
  e4m3x4_to_floats(*p, f);
  return f[0] * factor;
}

// One row by one warp on the CUDA cores: lane l holds dimensions l, l + 32, ...
// (N of them); the keys it sees, and no others, are walked one by one with a
// running maximum and sum in fp32.  Head sizes that the tensor-core kernels do
// not take run on this; and those kernels call it for a row that came out
// infinite or NaN while some of its piece's keys are hidden from it: a matrix
// product multiplies a hidden key's value by 0, which an infinity or a NaN in
// it survives.
template <typename T, typename KV, int N>
__device__ void attend_row(const Problem& p, int64_t tok, int head) {
  const int lane = threadIdx.x & 31;
  const int kvh = head / (p.heads / p.kv_heads);
  const int D = p.head_dim;
  const T* q = static_cast<const T*>(p.query) + tok * p.q_stride + (int64_t)head * D;
  const KV* cache = static_cast<const KV*>(p.cache);
  const TokenInfo info = p.tokens[tok];
  float qv[N], acc[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int d = lane + 32 * i;
    qv[i] = d < D ? Traits<T>::to_f(q[d]) : 0.f;
    acc[i] = 0.f;
  }
  const float slope = p.slopes ? p.slopes[head] : 0.f;
  const uint64_t* bits = p.tree_mask ? p.tree_mask + tok * p.tree_words : nullptr;
  const int end = bits ? info.pos : info.hi;  // a tree's drafted keys are hi .. pos - 1
  float m = -INFINITY, l = 0.f;
  for (int j = info.lo; j < end; ++j) {
    if (j >= info.hi && !tree_bit(bits, j - info.hi)) continue;
    const int64_t page = p.kv_indices[info.page_base + page_number(p, j)];
    const int64_t krow = (page * 2 * p.page_size + page_slot(p, j)) * p.kv_heads + kvh;
    const int64_t vrow = krow + (int64_t)p.page_size * p.kv_heads;
    float kf = 1.f, vf = 1.f;
    if (p.exponents) {
      kf = exponent_factor(p.exponents[krow]);
      vf = exponent_factor(p.exponents[vrow]);
    }
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int d = lane + 32 * i;
      if (d < D) dot += qv[i] * load_kv(cache + krow * D + d, kf);
    }
    for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    const float s = score(dot, p.scale, p.cap, slope, abs(info.pos - j));
    const float m2 = fmaxf(m, s);  // a NaN stays out of the maximum and enters the sum
    const float c = m2 == -INFINITY ? 1.f : expf(m - m2);
    const float e = s == -INFINITY ? 0.f : expf(s - m2);
    l = l * c + e;
    m = m2;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int d = lane + 32 * i;
      if (d < D) acc[i] = acc[i] * c + e * load_kv(cache + vrow * D + d, vf);
    }
  }
  T* o = static_cast<T*>(p.out) + tok * p.out_stride + (int64_t)head * D;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int d = lane + 32 * i;
    if (d < D) o[d] = Traits<T>::from_f(l == 0.f ? 0.f : acc[i] / l);
  }
  if (p.lse && lane == 0) p.lse[tok * p.heads + head] = l == 0.f ? -INFINITY : m + logf(l);
}

}  // namespace attn
}  // namespace pace
