// A step's page tables and index arrays from its requests' lengths, for
// sm_100a: what PaceServe's block manager and attention wrapper build on the
// host (flashinfer_attention_wrapper.py:75-209) and copy to the device.
//
// Request b holds ceil(seq_b / page) pages, the first of its row of the block
// table, and gets new_b tokens more.  New pages come from the top of a stack of
// free ones, in the requests' order: the k-th is free[count - 1 - k].  All else
// follows from three prefix sums over the requests (new tokens, pages, new
// pages).  Every CTA works them out for itself (they are a few KB, from L2) and
// then takes its share of the outputs, finding an entry's request by bisection
// in shared memory; so one launch does without a grid-wide barrier.  The two
// values that are read by all and changed, the stack's height and the status, are
// written by the CTA that read them last.  It is a matter of latency: a few
// dependent loads.
//
// Lengths that moved on after a step that did not fit would count pages as held
// that were never given: their entries of the block table are an earlier owner's.
// So a call does nothing while the status is set.
#include <algorithm>

#include "common.cuh"

namespace pace {
namespace {

constexpr int kThreads = 512;  // at most
constexpr int64_t kMaxRequests = 8192;  // three prefix sums of them in shared memory

struct TableJob {
  int32_t* block_tables;
  const int32_t *lens_a, *lens_b;  // build: in the cache, new;  release: held, kept
  int32_t *free_pages, *free_count;
  int32_t *append_indptr, *kv_indptr, *kv_indices, *last_page_len, *batch_indices;
  int64_t *positions, *slots;
  int32_t *status, *arrivals;
  int64_t table_stride, max_blocks, num_free_pages, num_indices, num_tokens;
  int requests, page_size, page_shift;
  int no_bits;  // 0, which the compiler does not know
};

__device__ __forceinline__ int64_t pages_of(const TableJob& j, int64_t tokens) {
  const int64_t t = tokens + j.page_size - 1;
  return j.page_shift >= 0 ? t >> j.page_shift : t / j.page_size;
}

// Sums stop at this, far above any array: they are compared with the arrays'
// lengths, and adding without overflow stays associative.
constexpr uint32_t kTooMany = 0x7fffffffu;
__device__ __forceinline__ uint32_t add(uint32_t a, uint32_t b) { return min(a + b, kTooMany); }

// Exclusive prefix sums of three values over the CTA; totals in `all`.
__device__ __forceinline__ void scan3(uint32_t (&v)[3], uint32_t (&all)[3], uint32_t (*part)[3]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  auto inclusive = [&](uint32_t (&x)[3]) {
#pragma unroll
    for (int d = 1; d < 32; d <<= 1)
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        const uint32_t o = __shfl_up_sync(0xffffffffu, x[k], d);
        if (lane >= d) x[k] = add(x[k], o);
      }
  };
  uint32_t before[3], mine[3], w[3];
  inclusive(v);
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    if (lane == 31) part[warp][k] = v[k];
    before[k] = __shfl_up_sync(0xffffffffu, v[k], 1);
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 3; ++k) w[k] = lane < warps ? part[lane][k] : 0u;
  inclusive(w);  // by every warp
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    all[k] = __shfl_sync(0xffffffffu, w[k], 31);
    mine[k] = __shfl_sync(0xffffffffu, w[k], max(warp - 1, 0));
    v[k] = add(lane ? before[k] : 0u, warp ? mine[k] : 0u);
  }
}

// The request whose range of an ascending prefix sum holds `i`.
__device__ __forceinline__ int owner_of(const int32_t* sum, int requests, int i) {
  int lo = 0, hi = requests - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (sum[mid] <= i)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

// BUILD: a step's arrays; otherwise pages go back onto the stack.
template <bool BUILD>
__global__ void __launch_bounds__(kThreads) step_tables_kernel(const TableJob j) {
  extern __shared__ int32_t sums[];  // [requests + 1] each: first, pages, new pages
  __shared__ uint32_t part[32][3];
  __shared__ int problem_bits, height_read, status_read;
  const int R = j.requests, threads = blockDim.x;
  int32_t* ip = sums;              // BUILD: new tokens; release: pages kept
  int32_t* kp = sums + R + 1;      // BUILD: pages
  int32_t* np = sums + 2 * R + 2;  // BUILD: new pages; release: pages given back
  pdl_launch_dependents();
  pdl_wait();
  // The stack's height and the status are read once a CTA.  The CTA that has read them last writes the
  // new ones: what an arrival adds is made from both (of no bit of them), so it is issued when they
  // have come, and when the last one has counted, every CTA has its own.
  uint32_t before = 0;
  if (threadIdx.x == 0) {
    problem_bits = 0;
    const int32_t h = *reinterpret_cast<volatile int32_t*>(j.free_count);
    const int32_t set = *reinterpret_cast<volatile int32_t*>(j.status);
    height_read = h;
    status_read = set;
    if (gridDim.x > 1) before = atomicAdd(j.arrivals, 1 + ((h | set) & j.no_bits));
  }
  auto leave = [&](int64_t height, int32_t problems) {
    if (threadIdx.x != 0 || before != gridDim.x - 1) return;
    if (gridDim.x > 1) *j.arrivals = 0;
    if (problems)
      atomicOr(j.status, problems);
    else
      *j.free_count = (int32_t)height;
  };
  uint32_t v[3] = {0, 0, 0}, all[3];
  int32_t problems = 0;
  // what request b adds to the three sums
  auto shares = [&](int b, uint32_t (&s)[3]) {
    const int64_t x = j.lens_a[b], y = j.lens_b[b];
    const int64_t most = BUILD ? x + y : x;
    if (x < 0 || y < 0 || (!BUILD && y > x)) {
      problems |= PACE_TABLES_BAD_LENGTH;
      s[0] = s[1] = s[2] = 0;
      return;
    }
    // pages at most 2^32: as many as fit a sum
    const int64_t pages = pages_of(j, most), less = pages_of(j, BUILD ? x : y);
    if (pages > j.max_blocks) problems |= PACE_TABLES_SHORT_ROW;
    s[0] = BUILD ? (uint32_t)y : 0u;
    s[1] = BUILD ? (uint32_t)min(pages, (int64_t)kTooMany) : 0u;
    s[2] = (uint32_t)min(pages - less, (int64_t)kTooMany);
  };
  for (int b = threadIdx.x; b < R; b += threads) {
    shares(b, v);
    // release keeps what its rows begin with in ip
    ip[b] = BUILD ? v[0] : (int32_t)pages_of(j, j.lens_b[b]);
    kp[b] = v[1];
    np[b] = v[2];
  }
  // a thread's requests: the one it has, or neighbours, an odd number of them, so that a warp's
  // threads use different banks
  const int per = (R + threads - 1) / threads | 1;
  const int b0 = min(R, (int)threadIdx.x * per), b1 = min(R, b0 + per);
  if (per > 1) {
    __syncthreads();
    v[0] = v[1] = v[2] = 0;
    for (int b = b0; b < b1; ++b) {
      if (BUILD) {
        v[0] = add(v[0], ip[b]);
        v[1] = add(v[1], kp[b]);
      }
      v[2] = add(v[2], np[b]);
    }
  }
  scan3(v, all, part);
  const int64_t height = height_read;
  if (BUILD) {
    if (all[1] > j.num_indices || all[1] == kTooMany) problems |= PACE_TABLES_SHORT_INDICES;
    if (all[0] > j.num_tokens || all[0] == kTooMany) problems |= PACE_TABLES_SHORT_TOKENS;
    if (height < 0 || height > j.num_free_pages || all[2] > height || all[2] == kTooMany)
      problems |= PACE_TABLES_NO_PAGES;
  } else if (height < 0 || height + all[2] > j.num_free_pages || all[2] == kTooMany) {
    problems |= PACE_TABLES_NO_PAGES;
  }
  if (problems) atomicOr(&problem_bits, problems);
  __syncthreads();
  problems = status_read ? status_read : problem_bits;  // the first cause stays the only one
  const int64_t step = (int64_t)gridDim.x * threads;
  const int64_t me = (int64_t)blockIdx.x * threads + threadIdx.x;
  if (problems) {
    // nothing is taken or given; tables that no token gets through
    if (BUILD) {
      for (int64_t i = me; i <= R; i += step) {
        j.append_indptr[i] = j.kv_indptr[i] = 0;
        if (i < R) j.last_page_len[i] = 0;
      }
      for (int64_t i = me; i < j.num_tokens; i += step) {
        j.batch_indices[i] = -1;
        j.positions[i] = j.slots[i] = -1;
      }
    }
    leave(height, problems);
    return;
  }
  for (int b = b0; b < b1; ++b) {
    auto place = [&](int32_t* sum, uint32_t& at) {
      const uint32_t share = sum[b];
      sum[b] = (int32_t)at;
      at = add(at, share);
    };
    if (BUILD) {
      place(ip, v[0]);
      place(kp, v[1]);
    }
    place(np, v[2]);
  }
  if (threadIdx.x == 0) {
    ip[R] = (int32_t)all[0];
    kp[R] = (int32_t)all[1];
    np[R] = (int32_t)all[2];
  }
  __syncthreads();
  if constexpr (BUILD) {
    // page k of request b, old or new
    auto page_at = [&](int b, int k, bool* fresh) -> int32_t {
      const int held = (kp[b + 1] - kp[b]) - (np[b + 1] - np[b]);
      *fresh = k >= held;
      return *fresh ? j.free_pages[height - 1 - (np[b] + k - held)]
                    : j.block_tables[(int64_t)b * j.table_stride + k];
    };
    for (int64_t i = me; i <= R; i += step) {
      j.append_indptr[i] = ip[i];
      j.kv_indptr[i] = kp[i];
      if (i < R) {
        // 1 .. page_size; page_size for a request without tokens, whose length is then 0
        const int64_t n = (int64_t)j.lens_a[i] + j.lens_b[i];
        j.last_page_len[i] = (int32_t)(n - (pages_of(j, n) - 1) * j.page_size);
      }
    }
    const int pages = (int)all[1], tokens = (int)all[0];
    // a warp takes 256 neighbouring pages: each lane has all its loads under way before the first
    // store, and looks a page's request up only where it is another than the last one's
    constexpr int kEach = 8;
    const int64_t chunk = kEach * 32, chunks_step = step / 32 * chunk;
    const int64_t mine = me / 32 * chunk + (threadIdx.x & 31);
    for (int64_t i0 = mine; i0 < pages; i0 += chunks_step) {
      int b = owner_of(kp, R, (int)i0);
      int32_t page[kEach];
      int32_t* entry[kEach];  // of the block table, for a new page
#pragma unroll
      for (int u = 0; u < kEach; ++u) {
        const int64_t i = i0 + u * 32;
        entry[u] = nullptr;
        if (i >= pages) continue;
        if (kp[b + 1] <= (int)i) b = owner_of(kp, R, (int)i);
        const int k = (int)i - kp[b];
        bool fresh;
        page[u] = page_at(b, k, &fresh);
        if (fresh) entry[u] = j.block_tables + (int64_t)b * j.table_stride + k;
      }
#pragma unroll
      for (int u = 0; u < kEach; ++u) {
        const int64_t i = i0 + u * 32;
        if (i < pages) j.kv_indices[i] = page[u];
        if (entry[u]) *entry[u] = page[u];
      }
    }
    // tokens from the other end of the grid: its first CTAs have pages
    for (int64_t i = step - 1 - me; i < j.num_tokens; i += step) {
      int64_t pos = -1, slot = -1;
      int b = -1;  // padding
      if (i < tokens) {
        b = owner_of(ip, R, (int)i);
        pos = (int64_t)j.lens_a[b] + ((int)i - ip[b]);
        const int k = (int)(j.page_shift >= 0 ? pos >> j.page_shift : pos / j.page_size);
        bool fresh;
        slot = (int64_t)page_at(b, k, &fresh) * j.page_size + (pos - (int64_t)k * j.page_size);
      }
      j.batch_indices[i] = b;
      j.positions[i] = pos;
      j.slots[i] = slot;
    }
    leave(height - all[2], 0);
  } else {
    const int given = (int)all[2];
    for (int64_t i = me; i < given; i += step) {
      const int b = owner_of(np, R, (int)i), k = ip[b] + ((int)i - np[b]);
      j.free_pages[height + given - 1 - i] = j.block_tables[(int64_t)b * j.table_stride + k];
    }
    leave(height + given, 0);
  }
}

template <bool BUILD>
int run_tables(TableJob& j, int64_t requests, int64_t page_size, cudaStream_t stream,
               const char* name) {
  if (requests < 0 || page_size <= 0 || page_size > INT32_MAX || j.max_blocks < 0 ||
      j.num_free_pages < 0 || j.num_indices < 0 || j.num_tokens < 0)
    return fail(PACE_ERR_INVALID_ARGUMENT, "%s: bad shape", name);
  if (requests > 1 && j.table_stride < j.max_blocks)
    return fail(PACE_ERR_INVALID_ARGUMENT, "%s: row stride smaller than the row", name);
  if (requests > kMaxRequests)
    return fail(PACE_ERR_TOO_LARGE, "%s: %lld requests, at most %lld", name, (long long)requests,
                (long long)kMaxRequests);
  if (j.num_free_pages > INT32_MAX || j.num_indices > INT32_MAX || j.num_tokens > INT32_MAX ||
      j.max_blocks > INT32_MAX)
    return fail(PACE_ERR_TOO_LARGE, "%s: index arrays longer than 2^31 - 1", name);
  if (!j.free_count || !j.status || !j.arrivals || (j.num_free_pages > 0 && !j.free_pages) ||
      (requests > 0 && (!j.lens_a || !j.lens_b || (j.max_blocks > 0 && !j.block_tables))) ||
      (BUILD && (!j.append_indptr || !j.kv_indptr || (requests > 0 && !j.last_page_len) ||
                 (j.num_indices > 0 && !j.kv_indices) ||
                 (j.num_tokens > 0 && (!j.batch_indices || !j.positions || !j.slots)))))
    return fail(PACE_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
  j.requests = (int)requests;
  j.page_size = (int)page_size;
  j.page_shift = (page_size & (page_size - 1)) == 0 ? __builtin_ctzll(page_size) : -1;
  StreamDeviceGuard guard(stream);
  const int smem = (int)(3 * (requests + 1) * sizeof(int32_t));
  cudaError_t err = cudaSuccess;
  if (smem > 48 * 1024) {
    err = ensure_dynamic_smem(reinterpret_cast<const void*>(step_tables_kernel<BUILD>),
                              guard.device(), (int)(3 * (kMaxRequests + 1) * sizeof(int32_t)));
    if (err != cudaSuccess) return cuda_fail(err, name);
  }
  // a few entries a thread, of the arrays' full length: how much of it a step needs is known on
  // the device only.  One CTA where they are few: it needs no arrival
  const int64_t entries = BUILD ? j.num_indices + j.num_tokens
                                : (j.max_blocks < 1 ? 0 : requests * j.max_blocks);
  const int threads = requests <= 128 && entries <= 1024 ? 128 : kThreads;
  const int64_t each = (BUILD ? 8 : 32) * threads;  // a release seldom gives all that rows can hold
  const int64_t ctas =
      std::min<int64_t>(sm_count(guard.device()), std::max<int64_t>(1, ceil_div(entries, each)));
  err = launch(step_tables_kernel<BUILD>, dim3((unsigned)ctas), dim3((unsigned)threads),
               (size_t)smem, stream, j);
  return err == cudaSuccess ? PACE_OK : cuda_fail(err, name);
}

}  // namespace
}  // namespace pace

extern "C" int pace_build_step_tables(
    int32_t* block_tables, int64_t table_row_stride, int64_t max_blocks, const int32_t* seq_lens,
    const int32_t* new_lens, int64_t num_requests, int64_t page_size, int32_t* free_pages,
    int64_t num_free_pages, int32_t* free_count, int32_t* append_indptr, int32_t* kv_indptr,
    int32_t* kv_indices, int64_t num_kv_indices, int32_t* kv_last_page_len,
    int32_t* batch_indices, int64_t* positions, int64_t* slot_mapping, int64_t num_tokens,
    int32_t* status, int32_t* arrivals, cudaStream_t stream) {
  pace::TableJob j = {};
  j.block_tables = block_tables;
  j.table_stride = table_row_stride;
  j.max_blocks = max_blocks;
  j.lens_a = seq_lens;
  j.lens_b = new_lens;
  j.free_pages = free_pages;
  j.num_free_pages = num_free_pages;
  j.free_count = free_count;
  j.append_indptr = append_indptr;
  j.kv_indptr = kv_indptr;
  j.kv_indices = kv_indices;
  j.num_indices = num_kv_indices;
  j.last_page_len = kv_last_page_len;
  j.batch_indices = batch_indices;
  j.positions = positions;
  j.slots = slot_mapping;
  j.num_tokens = num_tokens;
  j.status = status;
  j.arrivals = arrivals;
  return pace::run_tables<true>(j, num_requests, page_size, stream, "build_step_tables");
}

extern "C" int pace_release_pages(const int32_t* block_tables, int64_t table_row_stride,
                                  int64_t max_blocks, const int32_t* held_lens,
                                  const int32_t* kept_lens, int64_t num_requests,
                                  int64_t page_size, int32_t* free_pages, int64_t num_free_pages,
                                  int32_t* free_count, int32_t* status, int32_t* arrivals,
                                  cudaStream_t stream) {
  pace::TableJob j = {};
  j.block_tables = const_cast<int32_t*>(block_tables);
  j.table_stride = table_row_stride;
  j.max_blocks = max_blocks;
  j.lens_a = held_lens;
  j.lens_b = kept_lens;
  j.free_pages = free_pages;
  j.num_free_pages = num_free_pages;
  j.free_count = free_count;
  j.status = status;
  j.arrivals = arrivals;
  return pace::run_tables<false>(j, num_requests, page_size, stream, "release_pages");
}
