// Paged KV cache addressing shared by the append, quantised append and read
// back kernels: [num_pages, 2, page_size, kv_heads, head_dim] pages found
// through kv_indptr / kv_indices / kv_last_page_len.
#pragma once

#include "common.cuh"

namespace pace {

// Requests whose per-request metadata (append_indptr, kv_indptr,
// kv_last_page_len) each CTA stages in shared memory: 3 x 2049 x 4 B.
constexpr int64_t kMaxStagedBatch = 2048;

struct PageTable {
  int64_t num_pages;
  int page_size;
  int64_t batch;
  int64_t num_indices;  // entries of kv_indices
};

// Page and slot of a token of request b at sequence position pos, or false
// if any index is out of range.  ip / last: kv_indptr and kv_last_page_len
// (global or staged copies).  A last-page length outside [1, page_size] makes
// the request's length inconsistent with its page count, so its tokens are
// rejected rather than placed on a page past the request's range.
__device__ __forceinline__ bool locate_token(const PageTable& j, int b, int64_t pos,
                                             const int32_t* kv_indices, const int32_t* ip,
                                             const int32_t* last, int64_t* page, int* slot) {
  if (b < 0 || b >= j.batch || pos < 0) return false;
  const int64_t p0 = ip[b];
  const int64_t np = (int64_t)ip[b + 1] - p0;
  if (np <= 0 || p0 < 0 || p0 + np > j.num_indices) return false;
  const int64_t lp = last[b];
  if (lp < 1 || lp > j.page_size) return false;
  const int64_t seq_len = (np - 1) * j.page_size + lp;
  if (pos >= seq_len) return false;  // so pos / page_size < np
  const int64_t pg = kv_indices[p0 + pos / j.page_size];
  if (pg < 0 || pg >= j.num_pages) return false;
  *page = pg;
  *slot = (int)(pos % j.page_size);
  return true;
}

// Request of token i from append_indptr (ascending, batch + 1 entries).
__device__ __forceinline__ int find_request(const int32_t* indptr, int64_t batch, int64_t i) {
  int lo = 0, hi = (int)batch - 1;  // largest b with indptr[b] <= i
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (indptr[mid] <= i)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

}  // namespace pace
