// Paged attention: the plan of a step's work, the entry points, and the
// CUDA-core kernel that takes any head size.
//
// PaceServe runs attention through FlashInfer's paged wrappers: begin_forward
// plans a step once (paceserve/model_executor/attention/
// flashinfer_attention_wrapper.py:75-209), every layer then runs on the plan
// (:245-275).  The same split is kept here: pace_paged_attention_plan works on
// the host arrays of the step and writes records that every layer's
// pace_paged_attention reads on the device.
#include <string.h>

#include <algorithm>
#include <exception>
#include <vector>

#include "attention_mma.cuh"

namespace pace {
namespace attn {

constexpr int kMaxHeadDim = 256;
constexpr int kWarps = 4;

// One warp per (query token, head).
template <typename T, typename KV>
__global__ void __launch_bounds__(kWarps * 32) attention_rows_kernel(const Problem p) {
  pdl_launch_dependents();
  pdl_wait();
  const int64_t w = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (w >= p.total_q * p.heads) return;
  attend_row<T, KV, kMaxHeadDim / 32>(p, w / p.heads, (int)(w % p.heads));
}

template <typename T, typename KV>
int run_rows(const Problem& p, cudaStream_t stream, const char* what) {
  const int64_t warps = p.total_q * p.heads;
  const cudaError_t err =
      launch(attention_rows_kernel<T, KV>, dim3((unsigned)ceil_div(warps, kWarps)),
             dim3(kWarps * 32), 0, stream, p);
  return err == cudaSuccess ? PACE_OK : cuda_fail(err, what);
}

// ---------------------------------------------------------------- the plan --
// Query rows (tokens x heads per kv head) one piece of the few-row kernel and
// of the tile kernel takes.  64 draft trees of up to 4 tokens (16 rows) over up to
// 4500 take 101 us in the former; of up to 8 (32 rows), mostly in the latter, 164.
constexpr int kFewRows = 16;
constexpr int kTileRows = 256;
// Keys per step of the two kernels, the unit in which pieces are cut.
constexpr int kFewKeys = 64;
constexpr int kTileKeys = 128;
// A piece is not cut below this many units: each cut costs the writing and
// reading of a partial result (one token over 333: 7.9 us whole, 8.6 in pieces of
// 128 keys; a tree of 13 over 344: 13.3 whole, 16.0 in pieces of 128).
constexpr int kFewMinUnits = 4;
constexpr int kTileMinUnits = 4;
// Pieces per CTA slot that the cutting aims at; the hardware hands them out
// longest first, so more of them even out ragged lengths better, but each pays for
// its start and its partial result.  Measured, 1 / 2 / 3 pieces: 64 decode requests
// 197 / 210 / 207 us, 32 draft trees over a quantised cache 133 / 176 / 196 us.
constexpr int kPiecesPerSlot = 1;
constexpr int kFewCtasPerSm = 2;

// Counters at the head of the workspace.  Their place must not move from plan to
// plan: every launch leaves them zero, what lies behind them not.
constexpr int kCounters = 16384;

// Cuts pieces longer than the even share of a slot, at most max_tiles of them,
// and orders all longest first.  Returns the number of partial slots used.
int cut_items(std::vector<Item>& items, int unit, int min_units, int64_t slots, int max_tiles,
              int* tiles) {
  int64_t total = 0;
  // cuts lie on multiples of the unit, so that only a sequence's first step is ragged
  auto cost = [&](const Item& w) -> int64_t {
    return w.kv_end > w.kv_begin ? ceil_div(w.kv_end, unit) - w.kv_begin / unit : 0;
  };
  for (const Item& w : items) total += cost(w);
  const int64_t share = std::max<int64_t>(min_units, ceil_div(total, slots * kPiecesPerSlot));
  std::vector<Item> cut;
  cut.reserve(items.size() * 2);
  int slot = 0, tile = 0;
  for (Item w : items) {
    const int64_t n = cost(w);
    const int64_t parts = n > share + share / 2 && tile < max_tiles ? ceil_div(n, share) : 1;
    w.tile = 0;
    w.slot = 0;
    w.splits = (int)parts;
    if (parts > 1) {
      w.tile = tile++;
      w.slot = slot;
      slot += (int)parts;
    }
    const int begin = w.kv_begin, end = w.kv_end, base = begin / unit * unit;
    for (int64_t k = 0; k < parts; ++k) {
      w.split = (int)k;
      w.kv_begin = k > 0 ? base + (int)(n * k / parts) * unit : begin;
      w.kv_end = k + 1 < parts ? base + (int)(n * (k + 1) / parts) * unit : end;
      cut.push_back(w);
    }
  }
  std::stable_sort(cut.begin(), cut.end(),
                   [&](const Item& a, const Item& b) { return cost(a) > cost(b); });
  items.swap(cut);
  *tiles = tile;
  return slot;
}

// Words the plan may take: the tokens' records, kv_indices, and the items. A
// share is at least total / (slots * kPiecesPerSlot), so the cuts add at most
// that many items to the whole ones.
int64_t plan_capacity(int64_t batch, int64_t total_q, int64_t num_indices, int sms) {
  const int64_t slots = (int64_t)sms * kFewCtasPerSm * kPiecesPerSlot * 2;
  return 4 * total_q + num_indices + 12 * (2 * batch + total_q + slots) + 16;
}

// The workspace: counters, then the two kernels' partial rows (fp32) and their
// (maximum, sum) pairs, [slot][kv head][row].
struct Workspace {
  size_t few, few_ml, many, many_ml, bytes;
};

Workspace workspace_of(const pace_attention_plan& plan) {
  auto align = [](size_t n) { return (n + 255) & ~(size_t)255; };
  const size_t few = (size_t)plan.few_slots * plan.num_kv_heads * kFewRows;
  const size_t many = (size_t)plan.many_slots * plan.num_kv_heads * kTileRows;
  Workspace w;
  w.few = (size_t)kCounters * sizeof(int32_t);
  w.few_ml = align(w.few + few * plan.head_dim * sizeof(float));
  w.many = align(w.few_ml + few * sizeof(float2));
  w.many_ml = align(w.many + many * plan.head_dim * sizeof(float));
  w.bytes = align(w.many_ml + many * sizeof(float2));
  return w;
}

}  // namespace attn
}  // namespace pace

extern "C" int64_t pace_paged_attention_plan_words(int64_t batch_size, int64_t total_q,
                                                   int64_t num_kv_indices, int num_sms) {
  if (batch_size < 0 || total_q < 0 || num_kv_indices < 0 || num_sms <= 0) return 0;
  return pace::attn::plan_capacity(batch_size, total_q, num_kv_indices, num_sms);
}

extern "C" int pace_paged_attention_plan(
    pace_attention_plan* plan, int32_t* words, int64_t num_words, const int32_t* qo_indptr,
    const int32_t* kv_indptr, const int32_t* kv_indices, int64_t num_kv_indices,
    const int32_t* kv_last_page_len, int64_t batch_size, int num_heads, int num_kv_heads,
    int head_dim, int page_size, int window_left, const int32_t* prefix_lens,
    const int32_t* doc_starts, int tree_words, int num_sms) {
  using namespace pace;
  using namespace pace::attn;
  const char* what = "paged_attention_plan";
  if (!plan || batch_size < 0 || batch_size > (1 << 24) || num_kv_indices < 0 || page_size <= 0 ||
      num_sms <= 0 || tree_words < 0)
    return fail(PACE_ERR_INVALID_ARGUMENT, "%s: bad shape", what);
  if (num_kv_heads <= 0 || num_heads <= 0 || num_heads % num_kv_heads != 0 ||
      num_heads / num_kv_heads > 128 || num_kv_heads > 65535)
    return fail(PACE_ERR_INVALID_ARGUMENT,
                "%s: %d query heads over %d kv heads: a multiple of at most 128 is needed", what,
                num_heads, num_kv_heads);
  if (head_dim <= 0 || head_dim % 8 != 0 || head_dim > kMaxHeadDim)
    return fail(PACE_ERR_INVALID_ARGUMENT, "%s: head_dim %d must be a multiple of 8 up to %d", what,
                head_dim, kMaxHeadDim);
  if (tree_words > 0 && (window_left >= 0 || prefix_lens || doc_starts))
    return fail(PACE_ERR_INVALID_ARGUMENT, "%s: a tree takes no other mask", what);
  *plan = pace_attention_plan{};
  plan->batch_size = batch_size;
  plan->num_heads = num_heads;
  plan->num_kv_heads = num_kv_heads;
  plan->head_dim = head_dim;
  plan->page_size = page_size;
  plan->tree_words = tree_words;
  if (batch_size == 0) return PACE_OK;
  if (!words || !qo_indptr || !kv_indptr || !kv_last_page_len || (num_kv_indices > 0 && !kv_indices))
    return fail(PACE_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (qo_indptr[0] != 0 || kv_indptr[0] < 0)
    return fail(PACE_ERR_INVALID_ARGUMENT, "%s: qo_indptr must begin with 0 and kv_indptr not below",
                what);
  for (int64_t b = 0; b < batch_size; ++b) {
    const int64_t q = (int64_t)qo_indptr[b + 1] - qo_indptr[b];
    const int64_t pages = (int64_t)kv_indptr[b + 1] - kv_indptr[b];
    if (q < 0 || pages < 0 || kv_indptr[b + 1] > num_kv_indices)
      return fail(PACE_ERR_INVALID_ARGUMENT, "%s: indptr of request %lld is not ascending or passes "
                  "kv_indices", what, (long long)b);
    if (pages > 0 && (kv_last_page_len[b] < 1 || kv_last_page_len[b] > page_size))
      return fail(PACE_ERR_INVALID_ARGUMENT, "%s: kv_last_page_len %d of request %lld outside 1 .. %d",
                  what, kv_last_page_len[b], (long long)b, page_size);
    const int64_t len = pages > 0 ? (pages - 1) * page_size + kv_last_page_len[b] : 0;
    if (len > (1 << 30))
      return fail(PACE_ERR_TOO_LARGE, "%s: a sequence of %lld tokens", what, (long long)len);
    if (tree_words > 0 && (q > len || q > 64ll * tree_words))
      return fail(PACE_ERR_INVALID_ARGUMENT, "%s: request %lld drafts %lld tokens: at most its "
                  "length %lld and %d mask bits", what, (long long)b, (long long)q, (long long)len,
                  64 * tree_words);
    if (prefix_lens && prefix_lens[b] < 0)
      return fail(PACE_ERR_INVALID_ARGUMENT, "%s: negative prefix length", what);
  }
  const int64_t total_q = qo_indptr[batch_size];
  if (num_words < plan_capacity(batch_size, total_q, num_kv_indices, num_sms))
    return fail(PACE_ERR_INVALID_ARGUMENT, "%s: the plan needs %lld words", what,
                (long long)plan_capacity(batch_size, total_q, num_kv_indices, num_sms));
  int32_t max_page = -1;
  // the requests' entries; what lies before and behind them is not read
  for (int64_t i = kv_indptr[0]; i < kv_indptr[batch_size]; ++i) {
    if (kv_indices[i] < 0)
      return fail(PACE_ERR_INVALID_ARGUMENT, "%s: negative page in kv_indices", what);
    max_page = std::max(max_page, kv_indices[i]);
  }
  const int group = num_heads / num_kv_heads;
  const int tile_tokens = kTileRows / group;
  try {
    std::vector<Item> few, many;
    TokenInfo* tok = reinterpret_cast<TokenInfo*>(words);
    for (int64_t b = 0; b < batch_size; ++b) {
      const int q0 = qo_indptr[b], q = qo_indptr[b + 1] - q0;
      const int pages = kv_indptr[b + 1] - kv_indptr[b];
      const int len = pages > 0 ? (pages - 1) * page_size + kv_last_page_len[b] : 0;
      const bool is_few = (int64_t)q * group <= kFewRows;
      const int step = is_few ? q : tile_tokens;
      for (int t0 = 0; t0 < q; t0 += step) {
        const int n = std::min(step, q - t0);
        int first = len, end = 0;  // keys that some token of the piece sees
        bool mixed = tree_words > 0;  // a node may not even see itself
        for (int i = t0; i < t0 + n; ++i) {
          const int pos = len - q + i;
          TokenInfo& w = tok[q0 + i];
          int64_t lo = 0, hi = (int64_t)pos + 1;
          if (prefix_lens) hi = std::max<int64_t>(hi, prefix_lens[b]);
          if (window_left >= 0) lo = (int64_t)pos - window_left;
          if (doc_starts) lo = std::max<int64_t>(lo, doc_starts[q0 + i]);
          if (tree_words > 0) hi = len - q;
          lo = std::max<int64_t>(lo, 0);
          hi = std::min<int64_t>(hi, len);
          if (hi < lo) lo = hi = 0;
          w = TokenInfo{(int)lo, (int)hi, kv_indptr[b], tree_words > 0 ? len : pos};
          if (tree_words > 0) hi = len;
          if (hi > lo) {
            first = std::min(first, (int)lo);
            end = std::max(end, (int)hi);
          }
        }
        if (end <= first) first = end = 0;
        for (int i = t0; i < t0 + n && tree_words == 0; ++i)
          mixed |= tok[q0 + i].lo != first || tok[q0 + i].hi != end;
        Item w{};
        w.mixed = mixed;
        w.tok0 = q0 + t0;
        w.ntok = n;
        w.kv_begin = w.all_begin = first;
        w.kv_end = w.all_end = end;
        w.page_base = kv_indptr[b];
        (is_few ? few : many).push_back(w);
        if (is_few) plan->few_rows = std::max(plan->few_rows, n * group);
      }
    }
    const int64_t few_slots = (int64_t)ceil_div((int64_t)num_sms * kFewCtasPerSm, num_kv_heads);
    const int64_t many_slots = ceil_div(num_sms, num_kv_heads);
    const int max_tiles = kCounters / 2 / num_kv_heads;
    plan->few_slots =
        cut_items(few, kFewKeys, kFewMinUnits, few_slots, max_tiles, &plan->few_tiles);
    plan->many_slots =
        cut_items(many, kTileKeys, kTileMinUnits, many_slots, max_tiles, &plan->many_tiles);
    const Workspace ws = workspace_of(*plan);
    plan->workspace_bytes = ws.bytes;
    plan->total_q = total_q;
    plan->max_page = max_page;
    plan->num_few = (int)few.size();
    plan->num_many = (int)many.size();
    int64_t at = 4 * total_q;
    plan->few_offset = at;
    if (!few.empty()) memcpy(words + at, few.data(), few.size() * sizeof(Item));
    at += 12 * (int64_t)few.size();
    plan->many_offset = at;
    if (!many.empty()) memcpy(words + at, many.data(), many.size() * sizeof(Item));
    at += 12 * (int64_t)many.size();
    plan->indices_offset = at;
    if (num_kv_indices > 0) memcpy(words + at, kv_indices, (size_t)num_kv_indices * 4);
    at += num_kv_indices;
    plan->num_words = at;
  } catch (const std::exception& e) {
    return fail(PACE_ERR_INVALID_ARGUMENT, "%s: %s", what, e.what());
  }
  return PACE_OK;
}

extern "C" int pace_paged_attention(const pace_attention_plan* plan, const int32_t* plan_words,
                                    void* out, const void* query, int64_t query_token_stride,
                                    int64_t out_token_stride, const void* cache,
                                    const void* exponents, int64_t num_pages, float sm_scale,
                                    float logits_soft_cap, const float* alibi_slopes,
                                    const uint64_t* tree_mask, float* lse, void* workspace,
                                    size_t workspace_bytes, int32_t* fault_flags, int dtype,
                                    cudaStream_t stream) {
  using namespace pace;
  using namespace pace::attn;
  const char* what = "paged_attention";
  if (!plan || plan->total_q < 0)
    return fail(PACE_ERR_INVALID_ARGUMENT, "%s: no plan", what);
  const int64_t row = (int64_t)plan->num_heads * plan->head_dim;
  if (query_token_stride < row || out_token_stride < row)
    return fail(PACE_ERR_INVALID_ARGUMENT, "%s: token stride smaller than heads * head_dim", what);
  if (!(logits_soft_cap >= 0.f) || !(sm_scale == sm_scale))
    return fail(PACE_ERR_INVALID_ARGUMENT, "%s: logits_soft_cap must be 0 (none) or positive", what);
  if (plan->total_q == 0) return PACE_OK;
  if (plan->max_page >= num_pages)
    return fail(PACE_ERR_INVALID_ARGUMENT, "%s: kv_indices name page %d of a cache of %lld", what,
                plan->max_page, (long long)num_pages);
  if ((plan->tree_words > 0) != (tree_mask != nullptr))
    return fail(PACE_ERR_INVALID_ARGUMENT, "%s: a tree mask goes with a plan made for one", what);
  if (plan->tree_words > 0 && alibi_slopes)
    return fail(PACE_ERR_INVALID_ARGUMENT, "%s: a tree takes no distance bias", what);
  if (!plan_words || !out || !query || !cache)
    return fail(PACE_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  Problem p{};
  p.query = query;
  p.out = out;
  p.cache = cache;
  p.exponents = static_cast<const uint8_t*>(exponents);
  p.kv_indices = plan_words + plan->indices_offset;
  p.tokens = reinterpret_cast<const TokenInfo*>(plan_words);
  p.slopes = alibi_slopes;
  p.tree_mask = tree_mask;
  p.lse = lse;
  p.q_stride = query_token_stride;
  p.out_stride = out_token_stride;
  p.total_q = plan->total_q;
  p.heads = plan->num_heads;
  p.kv_heads = plan->num_kv_heads;
  p.head_dim = plan->head_dim;
  p.page_size = plan->page_size;
  p.tree_words = plan->tree_words;
  p.page_shift = -1;
  for (int s = 0; s < 31; ++s)
    if (plan->page_size == 1 << s) p.page_shift = s;
  p.scale = sm_scale;
  p.cap = logits_soft_cap < 1e30f ? logits_soft_cap : 0.f;  // such a cap bends no score
  // The tensor-core kernels take 16-bit queries of 64 or 128 dimensions over a cache that 16-byte
  // copies fit and whose rows 32 bits number; the CUDA-core kernel the rest.
  const int64_t cache_rows = num_pages * 2 * plan->page_size * plan->num_kv_heads;
  const bool tensor = (dtype == PACE_BF16 || dtype == PACE_F16) &&
                      (plan->head_dim == 64 || plan->head_dim == 128) && aligned16(cache) &&
                      cache_rows <= UINT32_MAX;
  // partial rows are written 32 bytes at a time
  if (tensor && (!workspace || workspace_bytes < plan->workspace_bytes ||
                 (reinterpret_cast<uintptr_t>(workspace) & 31) != 0))
    return fail(PACE_ERR_INVALID_ARGUMENT, "%s: the plan needs %zu bytes of 32-byte aligned "
                "workspace", what, plan->workspace_bytes);
  // a row that is done again reads its query once more
  if (out == query)
    return fail(PACE_ERR_INVALID_ARGUMENT, "%s: out must not be the query", what);
  StreamDeviceGuard guard(stream);
  if (tensor) {
    const Workspace ws = workspace_of(*plan);
    uint8_t* base = static_cast<uint8_t*>(workspace);
    int32_t* counters = reinterpret_cast<int32_t*>(base);
    const bool bf16 = dtype == PACE_BF16;
    if (plan->num_many > 0) {
      const int st = run_tile_rows(
          p, num_pages, reinterpret_cast<const Item*>(plan_words + plan->many_offset), plan->num_many,
          reinterpret_cast<float*>(base + ws.many), reinterpret_cast<float2*>(base + ws.many_ml),
          counters + kCounters / 2, fault_flags, bf16, guard.device(), stream, what);
      if (st != PACE_OK) return st;
    }
    if (plan->num_few == 0) return PACE_OK;
    return run_few_rows(p, plan->few_rows,
                        reinterpret_cast<const Item*>(plan_words + plan->few_offset),
                        plan->num_few, reinterpret_cast<float*>(base + ws.few),
                        reinterpret_cast<float2*>(base + ws.few_ml), counters, plan->num_many > 0,
                        bf16, guard.device(), stream, what);
  }
  return PACE_DISPATCH_FLOAT(dtype, what, [&] {
    using T = scalar_t;
    return exponents ? run_rows<T, uint8_t>(p, stream, what) : run_rows<T, T>(p, stream, what);
  });
}
