// The quantised paged KV cache for sm_100a: new K/V rows are quantised as they
// are appended, and a request's rows are read back in sequence order.
//
// The cache is two tensors per layer, both paged as PaceServe's 16-bit cache
// is (paceserve/model_executor/attention/flashinfer_attention_wrapper.py:53-73):
//   codes      [num_pages, 2, page_size, kv_heads, head_dim]  e4m3
//   exponents  [num_pages, 2, page_size, kv_heads]            one byte per row
// A row x (one token's K or V of one head) is held as
//   e = smallest integer >= -126 with max|x| <= 448 * 2^e,
//   code = e4m3(x * 2^-e) (nearest, ties to even), exponent = e + 127,
// where the scaling is exact, so each code has one rounding.  Infinities
// saturate at the largest code and do not enter the maximum; a row that holds
// a NaN gets exponent 255 and reads back as NaN.
//
// Both kernels move bytes and little else.  Append, per token: 4 * kv_heads *
// head_dim bytes of 16-bit input read, half of that plus 2 * kv_heads written.
#include "fp8.cuh"
#include "paged.cuh"

namespace pace {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxHeadDim = 256;

struct QuantJob : PageTable {
  int64_t rows;  // tokens appended or read back
  int heads;
  int head_dim;
  int64_t key_stride;
  int64_t value_stride;
  int lanes_log2;  // append: lanes (of 8 elements) per row, rounded up to a power of two
};

// Copies the per-request arrays to shared memory where they fit; the pointers
// are redirected to the copies.  A barrier follows before they are read.
__device__ __forceinline__ void stage_requests(const PageTable& t, int32_t* sh,
                                               const int32_t*& indptr, const int32_t*& kv_indptr,
                                               const int32_t*& last) {
  if (t.batch > kMaxStagedBatch) return;
  int32_t* s_ip = sh;
  int32_t* s_last = sh + t.batch + 1;
  int32_t* s_ai = sh + 2 * t.batch + 1;
  for (int64_t k = threadIdx.x; k <= t.batch; k += blockDim.x) {
    s_ip[k] = kv_indptr[k];
    if (k < t.batch) s_last[k] = last[k];
    s_ai[k] = indptr[k];
  }
  kv_indptr = s_ip;
  last = s_last;
  indptr = s_ai;
}

// Eight elements of a row as floats; elements at or past `valid` are zero.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, int valid, float* f) {
  if constexpr (VEC) {
    if (valid >= 8) {
      if constexpr (sizeof(T) == 4) {
        Traits<T>::unpack(ld_nc_v4(p), f);
        Traits<T>::unpack(ld_nc_v4(p + 4), f + 4);
      } else {
        Traits<T>::unpack(ld_nc_v4(p), f);
      }
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = i < valid ? Traits<T>::to_f(p[i]) : 0.f;
}

// One CTA: U tokens.  A row is quantised by a group of 2^lanes_log2 lanes, 8
// elements each; the maximum is a shuffle reduction, so every element is read
// once.  All of a pass's loads are issued before the token -> page lookups,
// which only the first U threads do.
template <typename T, int U, bool VEC>
__global__ void __launch_bounds__(kThreads)
    kv_quant_append_kernel(const T* __restrict__ key, const T* __restrict__ value,
                           const int32_t* __restrict__ append_indptr, uint8_t* __restrict__ codes,
                           uint8_t* __restrict__ exponents, const int32_t* __restrict__ kv_indices,
                           const int32_t* __restrict__ kv_indptr,
                           const int32_t* __restrict__ kv_last_page_len, QuantJob job,
                           int32_t* bad) {
  extern __shared__ int32_t sh[];
  __shared__ int64_t s_slot[U];  // K row slot of the token's page (V: + page_size), or -1
  pdl_launch_dependents();
  pdl_wait();
  const int64_t tok0 = (int64_t)blockIdx.x * U;
  const int ntok = (int)min((int64_t)U, job.rows - tok0);
  const int group = 1 << job.lanes_log2;
  const int rows_per_token = 2 * job.heads;
  const int units = (ntok * rows_per_token) << job.lanes_log2;
  const int32_t *ai = append_indptr, *ip = kv_indptr, *last = kv_last_page_len;
  for (int base = 0; base < units; base += U * kThreads) {
    float x[U][8];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int u = base + k * kThreads + (int)threadIdx.x;
      const int row = u >> job.lanes_log2;
      const int t = row / rows_per_token, kh = row - t * rows_per_token;
      const int c = (u & (group - 1)) * 8;
      const bool is_v = kh >= job.heads;
      const int valid = u < units ? job.head_dim - c : 0;  // <= 0: an idle lane
      const T* src = (is_v ? value + (tok0 + t) * job.value_stride
                           : key + (tok0 + t) * job.key_stride) +
                     (int64_t)(is_v ? kh - job.heads : kh) * job.head_dim + c;
      load8<T, VEC>(src, valid, x[k]);
    }
    if (base == 0) {
      stage_requests(job, sh, ai, ip, last);
      __syncthreads();
      if ((int)threadIdx.x < ntok) {
        const int64_t i = tok0 + threadIdx.x;
        const int b = find_request(ai, job.batch, i);
        int64_t page, at = -1;
        int slot;
        // i lies outside [ai[b], ai[b + 1]) where append_indptr does not cover it
        if (i >= (int64_t)ai[b] && i < (int64_t)ai[b + 1]) {
          const int64_t seq_len =
              ((int64_t)ip[b + 1] - ip[b] - 1) * job.page_size + last[b];
          const int64_t pos = seq_len - ai[b + 1] + i;
          if (locate_token(job, b, pos, kv_indices, ip, last, &page, &slot))
            at = page * 2 * job.page_size + slot;
        }
        s_slot[threadIdx.x] = at;
        if (at < 0 && bad) atomicAdd(bad, 1);
      }
      __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int u = base + k * kThreads + (int)threadIdx.x;
      float amax = 0.f;
      bool nan = false;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float a = fabsf(x[k][e]);
        nan |= a != a;
        if (a < INFINITY) amax = fmaxf(amax, a);
      }
      // NaN travels as a value above every finite magnitude
      if (nan) amax = INFINITY;
      for (int o = group >> 1; o > 0; o >>= 1)
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      const bool row_nan = amax == INFINITY;
      const uint32_t ex = row_nan ? (uint32_t)kNanExponent : row_exponent(amax);
      // 2^-e: an exact power of two, since e lies in [-126, 120]
      const float inv = row_nan ? 0.f : __uint_as_float((254u - ex) << 23);
      const int row = u >> job.lanes_log2;
      const int t = row / rows_per_token, kh = row - t * rows_per_token;
      const int c = (u & (group - 1)) * 8;
      if (u >= units || c >= job.head_dim) continue;
      const int64_t at = s_slot[t];
      if (at < 0) continue;
      const bool is_v = kh >= job.heads;
      const int64_t dst = (at + (is_v ? job.page_size : 0)) * job.heads + (is_v ? kh - job.heads : kh);
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = row_nan ? 0.f : x[k][e] * inv;
      const uint2 w = make_uint2(floats_to_e4m3x4(y), floats_to_e4m3x4(y + 4));
      *reinterpret_cast<uint2*>(codes + dst * job.head_dim + c) = w;
      if (c == 0) exponents[dst] = (uint8_t)ex;
    }
  }
}

// V codes' values times the row's factor, rounded once to T.
template <typename T, int V, bool VEC>
__device__ __forceinline__ void store_values(T* dst, const uint32_t (&codes)[V / 4], float factor) {
  float f[V];
#pragma unroll
  for (int i = 0; i < V / 4; ++i) e4m3x4_to_floats(codes[i], f + 4 * i);
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] *= factor;
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < V; i += Traits<T>::kVec) st_v4(dst + i, Traits<T>::pack(f + i));
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) dst[i] = Traits<T>::from_f(f[i]);
  }
}

// One CTA: `tokens` output rows (K and V of every head), V codes per thread
// and step.  The rows' places are looked up by the first threads; then each
// thread issues its U code loads together.
template <typename T, int V, int U, bool VEC>
__global__ void __launch_bounds__(kThreads)
    kv_quant_read_kernel(T* __restrict__ key, T* __restrict__ value,
                         const int32_t* __restrict__ out_indptr, const uint8_t* __restrict__ codes,
                         const uint8_t* __restrict__ exponents,
                         const int32_t* __restrict__ kv_indices,
                         const int32_t* __restrict__ kv_indptr,
                         const int32_t* __restrict__ kv_last_page_len, QuantJob job, int tokens,
                         int32_t* bad) {
  extern __shared__ int32_t sh[];
  __shared__ int64_t s_slot[kThreads];
  pdl_launch_dependents();
  pdl_wait();
  const int64_t tok0 = (int64_t)blockIdx.x * tokens;
  const int ntok = (int)min((int64_t)tokens, job.rows - tok0);
  const int32_t *oi = out_indptr, *ip = kv_indptr, *last = kv_last_page_len;
  stage_requests(job, sh, oi, ip, last);
  __syncthreads();
  if ((int)threadIdx.x < ntok) {
    const int64_t i = tok0 + threadIdx.x;
    const int b = find_request(oi, job.batch, i);
    int64_t page, at = -1;
    int slot;
    if (i >= (int64_t)oi[b] && i < (int64_t)oi[b + 1] &&
        locate_token(job, b, i - oi[b], kv_indices, ip, last, &page, &slot))
      at = page * 2 * job.page_size + slot;
    s_slot[threadIdx.x] = at;
    if (at < 0 && bad) atomicAdd(bad, 1);
  }
  __syncthreads();
  const int per_row = job.head_dim / V;
  const int per_token = 2 * job.heads * per_row;
  const int units = ntok * per_token;
  for (int base = 0; base < units; base += U * kThreads) {
    uint32_t w[U][V / 4];
    uint32_t ex[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int u = base + k * kThreads + (int)threadIdx.x;
      const int t = u / per_token, r = u - t * per_token;
      const int kh = r / per_row, c = (r - kh * per_row) * V;
      const int64_t at = u < units ? s_slot[t] : -1;
      ex[k] = 0;
#pragma unroll
      for (int i = 0; i < V / 4; ++i) w[k][i] = 0;
      if (at >= 0) {
        const bool is_v = kh >= job.heads;
        const int64_t src =
            (at + (is_v ? job.page_size : 0)) * job.heads + (is_v ? kh - job.heads : kh);
        const uint8_t* p = codes + src * job.head_dim + c;
        if constexpr (V == 16) {
          const uint4 q = ld_nc_v4(p);
          w[k][0] = q.x;
          w[k][1] = q.y;
          w[k][2] = q.z;
          w[k][3] = q.w;
        } else {
          const uint2 q = __ldg(reinterpret_cast<const uint2*>(p));
          w[k][0] = q.x;
          w[k][1] = q.y;
        }
        ex[k] = __ldg(exponents + src);
      }
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int u = base + k * kThreads + (int)threadIdx.x;
      if (u >= units) continue;
      const int t = u / per_token, r = u - t * per_token;
      const int kh = r / per_row, c = (r - kh * per_row) * V;
      if (s_slot[t] < 0) continue;
      const bool is_v = kh >= job.heads;
      T* dst = (is_v ? value + (tok0 + t) * job.value_stride : key + (tok0 + t) * job.key_stride) +
               (int64_t)(is_v ? kh - job.heads : kh) * job.head_dim + c;
      store_values<T, V, VEC>(dst, w[k], exponent_factor(ex[k]));
    }
  }
}

// Checks shared by the two entry points; PACE_OK with rows == 0 means nothing
// is to be done.
int check_job(const char* what, const void* key, const void* value, int64_t rows, int heads,
              int head_dim, int64_t key_stride, int64_t value_stride, const int32_t* indptr,
              const void* codes, const void* exponents, int64_t num_pages, int page_size,
              const int32_t* kv_indices, const int32_t* kv_indptr, const int32_t* last,
              int64_t batch) {
  if (rows < 0 || rows > INT32_MAX || heads <= 0 || heads > 4096 || page_size <= 0 ||
      num_pages < 0 || batch < 0)
    return fail(PACE_ERR_INVALID_ARGUMENT, "%s: bad shape", what);
  if (head_dim <= 0 || head_dim % 8 != 0 || head_dim > kMaxHeadDim)
    return fail(PACE_ERR_INVALID_ARGUMENT, "%s: head_dim %d must be a multiple of 8 up to %d", what,
                head_dim, kMaxHeadDim);
  const int64_t row = (int64_t)heads * head_dim;
  if (key_stride < row || value_stride < row)
    return fail(PACE_ERR_INVALID_ARGUMENT, "%s: row stride smaller than kv_heads * head_dim", what);
  if (rows == 0) return PACE_OK;
  if (batch == 0) return fail(PACE_ERR_INVALID_ARGUMENT, "%s: tokens but no requests", what);
  if (!key || !value || !indptr || !codes || !exponents || !kv_indices || !kv_indptr || !last)
    return fail(PACE_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (!aligned16(codes))
    return fail(PACE_ERR_INVALID_ARGUMENT, "%s: codes must be 16-byte aligned", what);
  return PACE_OK;
}

}  // namespace
}  // namespace pace

extern "C" int pace_append_quantised_paged_kv_cache(
    const void* key, const void* value, int64_t nnz, int num_kv_heads, int head_dim,
    int64_t key_row_stride, int64_t value_row_stride, const int32_t* append_indptr, void* codes,
    void* exponents, int64_t num_pages, int page_size, const int32_t* kv_indices,
    int64_t num_kv_indices, const int32_t* kv_indptr, const int32_t* kv_last_page_len,
    int64_t batch_size, int32_t* bad_tokens, int dtype, cudaStream_t stream) {
  using namespace pace;
  const char* what = "append_quantised_paged_kv_cache";
  const int st = check_job(what, key, value, nnz, num_kv_heads, head_dim, key_row_stride,
                           value_row_stride, append_indptr, codes, exponents, num_pages, page_size,
                           kv_indices, kv_indptr, kv_last_page_len, batch_size);
  if (st != PACE_OK || nnz == 0) return st;
  StreamDeviceGuard guard(stream);
  int lanes_log2 = 0;
  while ((8 << lanes_log2) < head_dim) ++lanes_log2;
  const QuantJob job{{num_pages, page_size, batch_size, num_kv_indices}, nnz, num_kv_heads, head_dim,
                     key_row_stride, value_row_stride, lanes_log2};
  const size_t smem = batch_size <= kMaxStagedBatch ? (size_t)(3 * batch_size + 2) * 4 : 0;
  const int sms = sm_count(guard.device());
  return PACE_DISPATCH_FLOAT(dtype, what, [&] {
    using T = scalar_t;
    constexpr int V = Traits<T>::kVec;
    const bool vec = key_row_stride % V == 0 && value_row_stride % V == 0 && aligned16(key) &&
                     aligned16(value);
    auto go = [&](auto kernel, int per_cta) {
      return launch(kernel, dim3((unsigned)ceil_div(nnz, per_cta)), dim3(kThreads), smem, stream,
                    static_cast<const T*>(key), static_cast<const T*>(value), append_indptr,
                    static_cast<uint8_t*>(codes), static_cast<uint8_t*>(exponents), kv_indices,
                    kv_indptr, kv_last_page_len, job, bad_tokens);
    };
    cudaError_t err;
    if (!vec)
      err = go(kv_quant_append_kernel<T, 1, false>, 1);
    else if (nnz <= 16 * sms)
      err = go(kv_quant_append_kernel<T, 1, true>, 1);
    else
      err = go(kv_quant_append_kernel<T, 4, true>, 4);
    if (err != cudaSuccess) return cuda_fail(err, what);
    return (int)PACE_OK;
  });
}

extern "C" int pace_read_quantised_paged_kv_cache(
    void* key, void* value, int64_t rows, int num_kv_heads, int head_dim, int64_t key_row_stride,
    int64_t value_row_stride, const int32_t* out_indptr, const void* codes, const void* exponents,
    int64_t num_pages, int page_size, const int32_t* kv_indices, int64_t num_kv_indices,
    const int32_t* kv_indptr, const int32_t* kv_last_page_len, int64_t batch_size,
    int32_t* bad_tokens, int dtype, cudaStream_t stream) {
  using namespace pace;
  const char* what = "read_quantised_paged_kv_cache";
  const int st = check_job(what, key, value, rows, num_kv_heads, head_dim, key_row_stride,
                           value_row_stride, out_indptr, codes, exponents, num_pages, page_size,
                           kv_indices, kv_indptr, kv_last_page_len, batch_size);
  if (st != PACE_OK || rows == 0) return st;
  StreamDeviceGuard guard(stream);
  const QuantJob job{{num_pages, page_size, batch_size, num_kv_indices}, rows, num_kv_heads,
                     head_dim, key_row_stride, value_row_stride, 0};
  const size_t smem = batch_size <= kMaxStagedBatch ? (size_t)(3 * batch_size + 2) * 4 : 0;
  const int sms = sm_count(guard.device());
  return PACE_DISPATCH_FLOAT(dtype, what, [&] {
    using T = scalar_t;
    constexpr int V = Traits<T>::kVec;
    const bool vec = key_row_stride % V == 0 && value_row_stride % V == 0 && aligned16(key) &&
                     aligned16(value);
    const int codes_per = head_dim % 16 == 0 ? 16 : 8;
    const int per_token = 2 * num_kv_heads * (head_dim / codes_per);
    auto go = [&](auto kernel, int u) {
      int64_t tokens = (int64_t)u * kThreads / per_token;  // one pass of the CTA
      tokens = tokens < 1 ? 1 : tokens > kThreads ? kThreads : tokens;
      return launch(kernel, dim3((unsigned)ceil_div(rows, tokens)), dim3(kThreads), smem, stream,
                    static_cast<T*>(key), static_cast<T*>(value), out_indptr,
                    static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(exponents),
                    kv_indices, kv_indptr, kv_last_page_len, job, (int)tokens, bad_tokens);
    };
    const bool few = rows * per_token <= (int64_t)8 * kThreads * sms;
    cudaError_t err;
    if (!vec)
      err = codes_per == 16 ? go(kv_quant_read_kernel<T, 16, 1, false>, 1)
                            : go(kv_quant_read_kernel<T, 8, 1, false>, 1);
    else if (codes_per == 16)
      err = few ? go(kv_quant_read_kernel<T, 16, 1, true>, 1)
                : go(kv_quant_read_kernel<T, 16, 4, true>, 4);
    else
      err = go(kv_quant_read_kernel<T, 8, 4, true>, 4);
    if (err != cudaSuccess) return cuda_fail(err, what);
    return (int)PACE_OK;
  });
}
