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
// a NaN gets exponent 255 and reads back as NaN.  Infinities among zeros alone
// have e = 0.  A finite element never takes a code whose value its type does not
// hold (256 * 2^8 of float16, 256 * 2^120 of the others), but the one below it.
//
// Both kernels move bytes and little else.  Append, per token: 4 * kv_heads *
// head_dim bytes of 16-bit input read, half of that plus 2 * kv_heads written.
#include <string.h>

#include <type_traits>

#include "fp8.cuh"
#include "paged.cuh"

namespace pace {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxHeadDim = 256;
constexpr int kResident = 6;  // CTAs that an SM holds

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

// Eight elements of a row as they are; elements at or past `valid` are zero.
template <typename T, bool VEC>
struct Raw8 {
  uint4 v[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p, int valid) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = make_uint4(0, 0, 0, 0);
    if (valid <= 0) return;
    if constexpr (VEC) {  // head_dim is a multiple of 8: all of them or none
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = ld_nc_v4(p + i * Traits<T>::kVec);
    } else {
      T e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = p[i];
      memcpy(v, e, sizeof(v));
    }
  }
};

// The exponent byte at which the type's largest magnitudes, from 248 * 2^e, would
// round to 256 * 2^e, which it does not hold: they take the code below it, 240, so
// that what was finite reads back finite.
template <typename T>
__device__ __forceinline__ constexpr uint32_t top_exponent() {
  return std::is_same<T, __half>::value ? 127 + 16 - 8 : 127 + 128 - 8;
}
__device__ __forceinline__ float below_256(float y) { return fminf(fmaxf(y, -240.f), 240.f); }

// Eight elements' codes and their row's exponent byte; the row is spread over
// `group` neighbouring lanes, all of which call.  In fp32, whatever the elements.
template <typename T>
__device__ __forceinline__ uint32_t quantise_floats(const float (&x)[8], int group, uint2& code) {
  float amax = 0.f;
  bool nan = false, inf = false;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float a = fabsf(x[e]);
    nan |= a != a;
    inf |= a == INFINITY;
    if (a < INFINITY) amax = fmaxf(amax, a);
  }
  // NaN travels as a value above every finite magnitude
  if (nan) amax = INFINITY;
  for (int o = group >> 1; o > 0; o >>= 1) {
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    inf |= __shfl_xor_sync(0xffffffffu, inf, o);
  }
  const bool row_nan = amax == INFINITY;
  // an infinity among zeros alone saturates at 448, not at 448 times next to nothing
  const uint32_t ex = row_nan               ? (uint32_t)kNanExponent
                      : inf && amax == 0.f ? 127u
                                           : row_exponent(amax);
  // 2^-e: an exact power of two, since e lies in [-126, 120]
  const float inv = row_nan ? 0.f : __uint_as_float((254u - ex) << 23);
  float y[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    y[e] = row_nan ? 0.f : x[e] * inv;
    if (ex == top_exponent<T>() && fabsf(x[e]) < INFINITY) y[e] = below_256(y[e]);
  }
  code = make_uint2(floats_to_e4m3x4(y), floats_to_e4m3x4(y + 4));
  return ex;
}

// The same from the elements' bits.  16-bit types find the maximum on pairs of
// magnitudes as integers; only a warp that holds an infinity, a NaN or one of the
// type's largest magnitudes takes the way above (which at 110 instructions for 8
// elements bound the kernel: 16167 fp16 tokens 39 us).
template <typename T>
__device__ __forceinline__ uint32_t quantise8(const uint4 (&v)[sizeof(T) / 2], int group,
                                              uint2& code) {
  float x[8];
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) Traits<T>::unpack(v[i], x + i * Traits<T>::kVec);
  if constexpr (sizeof(T) == 2) {
    constexpr uint32_t kMag = 0x7fff7fffu;
    uint32_t m = __vmaxu2(__vmaxu2(v[0].x & kMag, v[0].y & kMag),
                          __vmaxu2(v[0].z & kMag, v[0].w & kMag));
    for (int o = group >> 1; o > 0; o >>= 1)
      m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
    m = max(m & 0xffffu, m >> 16);
    // 248 * 2^e of the top exponent, past which lie infinities and NaN too
    constexpr uint32_t kTop = std::is_same<T, __half>::value ? 0x7bc0u : 0x7f78u;
    if (__all_sync(0xffffffffu, m < kTop)) {
      const uint16_t bits = (uint16_t)m;
      const uint32_t ex = row_exponent(Traits<T>::to_f(*reinterpret_cast<const T*>(&bits)));
      const float inv = __uint_as_float((254u - ex) << 23);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] *= inv;
      code = make_uint2(floats_to_e4m3x4(x), floats_to_e4m3x4(x + 4));
      return ex;
    }
  }
  return quantise_floats<T>(x, group, code);
}

// Where this thread works: as many tokens as fit the CTA side by side, `lanes`
// threads each; a token with more than kThreads units takes the CTA in turns.
constexpr int kMaxSide = kThreads / 4;  // of four rounds: a CTA looks up at most kThreads places
struct Place {
  int side;    // tokens side by side
  int sub;     // this thread's among them; >= side: idle
  int first;   // its first unit of the token
};
__device__ __forceinline__ Place place_of(int per_token) {
  if (per_token >= kThreads) return {1, 0, (int)threadIdx.x};
  Place p;
  p.side = min(kThreads / per_token, kMaxSide);
  p.sub = (int)threadIdx.x / per_token;
  p.first = (int)threadIdx.x - p.sub * per_token;
  return p;
}

// The tokens of a CTA: `batches` of U rounds of the tokens side by side.  A row is
// quantised by a group of 2^lanes_log2 lanes, 8 elements each; the maximum is a
// shuffle reduction, so every element is read once.  A batch's loads are issued
// before the batch in front of it is worked on, the first one's before the token
// -> page lookups, which the first threads do for all batches: the lookups are
// two loads that depend on each other, and with CTAs of one batch they were most
// of the time.  What bounds it is the loads in flight: 16167 fp16 tokens (103.6
// MB) take 25.6 us, 4.1 TB/s, in batches of two tokens with six CTAs an SM; 31 us
// in batches of four with four, 28 us in batches of one with eight, 39 us with one
// batch of four a CTA.  As float32 (172.5 MB) they take 44 us.
template <typename T, int U, bool VEC>
__global__ void __launch_bounds__(kThreads)
    kv_quant_append_kernel(const T* __restrict__ key, const T* __restrict__ value,
                           const int32_t* __restrict__ append_indptr, uint8_t* __restrict__ codes,
                           uint8_t* __restrict__ exponents, const int32_t* __restrict__ kv_indices,
                           const int32_t* __restrict__ kv_indptr,
                           const int32_t* __restrict__ kv_last_page_len, QuantJob job,
                           int batches, int32_t* bad) {
  extern __shared__ int32_t sh[];
  __shared__ int64_t s_slot[kThreads];  // K row slot of the token's page (V: + page_size), or -1
  const int group = 1 << job.lanes_log2;
  const int per_token = (2 * job.heads) << job.lanes_log2;
  const Place at = place_of(per_token);
  const int each = U * at.side;  // tokens of a batch
  const int64_t tok0 = (int64_t)blockIdx.x * each * batches;
  const int ntok = (int)min((int64_t)each * batches, job.rows - tok0);
  const int32_t *ai = append_indptr, *ip = kv_indptr, *last = kv_last_page_len;
  pdl_launch_dependents();
  pdl_wait();
  for (int base = 0; base < per_token; base += kThreads) {
    const int u = base + at.first;
    const int kh = u >> job.lanes_log2, c = (u & (group - 1)) * 8;
    const bool is_v = kh >= job.heads;
    const int head = is_v ? kh - job.heads : kh;
    const bool mine = at.sub < at.side && u < per_token && c < job.head_dim;
    const T* src = (is_v ? value : key) + (int64_t)head * job.head_dim + c;
    const int64_t stride = is_v ? job.value_stride : job.key_stride;
    Raw8<T, VEC> raw[U], next[U];
    auto load = [&](Raw8<T, VEC>(&r)[U], int t0) {
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int t = t0 + k * at.side + at.sub;
        r[k].load(src + (tok0 + t) * stride, mine && t < ntok ? 8 : 0);
      }
    };
    load(raw, 0);
    if (base == 0) {
      stage_requests(job, sh, ai, ip, last);
      __syncthreads();
      if ((int)threadIdx.x < ntok) {
        const int64_t i = tok0 + threadIdx.x;
        const int b = find_request(ai, job.batch, i);
        int64_t page, where = -1;
        int slot;
        // i lies outside [ai[b], ai[b + 1]) where append_indptr does not cover it
        if (i >= (int64_t)ai[b] && i < (int64_t)ai[b + 1]) {
          const int64_t seq_len =
              ((int64_t)ip[b + 1] - ip[b] - 1) * job.page_size + last[b];
          const int64_t pos = seq_len - ai[b + 1] + i;
          if (locate_token(job, b, pos, kv_indices, ip, last, &page, &slot))
            where = page * 2 * job.page_size + slot;
        }
        s_slot[threadIdx.x] = where;
        if (where < 0 && bad) atomicAdd(bad, 1);
      }
      __syncthreads();
    }
    for (int t0 = 0; t0 < ntok; t0 += each) {
      load(next, t0 + each);
#pragma unroll
      for (int k = 0; k < U; ++k) {
        uint2 code;
        const uint32_t ex = quantise8<T>(raw[k].v, group, code);
        const int t = t0 + k * at.side + at.sub;
        const int64_t where = mine && t < ntok ? s_slot[t] : -1;
        if (where >= 0) {
          const int64_t dst = (where + (is_v ? job.page_size : 0)) * job.heads + head;
          *reinterpret_cast<uint2*>(codes + dst * job.head_dim + c) = code;
          if (c == 0) exponents[dst] = (uint8_t)ex;
        }
      }
#pragma unroll
      for (int k = 0; k < U; ++k) raw[k] = next[k];
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
    constexpr int kVec = Traits<T>::kVec;
    if (V >= 2 * kVec && (reinterpret_cast<uintptr_t>(dst) & 31) == 0) {
#pragma unroll
      for (int i = 0; i < V / kVec; i += 2)
        st_v8(dst + i * kVec, Traits<T>::pack(f + i * kVec),
              Traits<T>::pack(f + (V >= 2 * kVec ? (i + 1) * kVec : 0)));
    } else {
#pragma unroll
      for (int i = 0; i < V; i += kVec) st_v4(dst + i, Traits<T>::pack(f + i));
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) dst[i] = Traits<T>::from_f(f[i]);
  }
}

// The output rows of a CTA: `batches` of U rounds of the tokens side by side, V
// codes per thread.  The rows' places are looked up by the first threads; a
// batch's loads are issued before the batch in front of it is written.  Memory
// bounds it: 23500 rows of K and V (192.9 MB) take 37.7 us, 5.1 TB/s.
template <typename T, int V, int U, bool VEC>
__global__ void __launch_bounds__(kThreads)
    kv_quant_read_kernel(T* __restrict__ key, T* __restrict__ value,
                         const int32_t* __restrict__ out_indptr, const uint8_t* __restrict__ codes,
                         const uint8_t* __restrict__ exponents,
                         const int32_t* __restrict__ kv_indices,
                         const int32_t* __restrict__ kv_indptr,
                         const int32_t* __restrict__ kv_last_page_len, QuantJob job, int batches,
                         int32_t* bad) {
  extern __shared__ int32_t sh[];
  __shared__ int64_t s_slot[kThreads];
  const int per_row = job.head_dim / V;
  const int per_token = 2 * job.heads * per_row;
  const Place at = place_of(per_token);
  const int each = U * at.side;  // tokens of a batch
  const int64_t tok0 = (int64_t)blockIdx.x * each * batches;
  const int ntok = (int)min((int64_t)each * batches, job.rows - tok0);
  const int32_t *oi = out_indptr, *ip = kv_indptr, *last = kv_last_page_len;
  pdl_launch_dependents();
  pdl_wait();
  stage_requests(job, sh, oi, ip, last);
  __syncthreads();
  if ((int)threadIdx.x < ntok) {
    const int64_t i = tok0 + threadIdx.x;
    const int b = find_request(oi, job.batch, i);
    int64_t page, where = -1;
    int slot;
    if (i >= (int64_t)oi[b] && i < (int64_t)oi[b + 1] &&
        locate_token(job, b, i - oi[b], kv_indices, ip, last, &page, &slot))
      where = page * 2 * job.page_size + slot;
    s_slot[threadIdx.x] = where;
    if (where < 0 && bad) atomicAdd(bad, 1);
  }
  __syncthreads();
  for (int u = at.first; u < per_token && at.sub < at.side; u += kThreads) {
    const int kh = u / per_row, c = (u - kh * per_row) * V;
    const bool is_v = kh >= job.heads;
    const int head = is_v ? kh - job.heads : kh;
    struct Codes {
      uint32_t w[V / 4];
      uint32_t ex;
      bool there;
    };
    Codes cur[U], next[U];
    auto load = [&](Codes(&r)[U], int t0) {
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int t = t0 + k * at.side + at.sub;
        const int64_t where = t < ntok ? s_slot[t] : -1;
        r[k].there = where >= 0;
        if (where >= 0) {
          const int64_t src = (where + (is_v ? job.page_size : 0)) * job.heads + head;
          const uint8_t* p = codes + src * job.head_dim + c;
          if constexpr (V == 16) {
            const uint4 q = ld_nc_v4(p);
            r[k].w[0] = q.x;
            r[k].w[1] = q.y;
            r[k].w[2] = q.z;
            r[k].w[3] = q.w;
          } else {
            const uint2 q = __ldg(reinterpret_cast<const uint2*>(p));
            r[k].w[0] = q.x;
            r[k].w[1] = q.y;
          }
          r[k].ex = __ldg(exponents + src);
        }
      }
    };
    T* dst = (is_v ? value : key) + (int64_t)head * job.head_dim + c;
    const int64_t stride = is_v ? job.value_stride : job.key_stride;
    load(cur, 0);
    for (int t0 = 0; t0 < ntok; t0 += each) {
      load(next, t0 + each);
#pragma unroll
      for (int k = 0; k < U; ++k) {
        if (cur[k].there)
          store_values<T, V, VEC>(dst + (tok0 + t0 + k * at.side + at.sub) * stride, cur[k].w,
                                  exponent_factor(cur[k].ex));
        cur[k] = next[k];
      }
    }
  }
}

// Tokens of a batch, and batches of a CTA: as many as leave every SM about
// `resident` CTAs, so that all run at once.
int64_t tokens_per_batch(int u, int per_token) {
  const int side = kThreads / per_token;
  return (int64_t)u * (side < 1 ? 1 : side > kMaxSide ? kMaxSide : side);
}
int batches_per_cta(int64_t rows, int64_t batch, int sms, int resident) {
  const int64_t n = ceil_div(rows, batch * sms * resident);
  const int64_t most = kThreads / batch;  // places that a CTA looks up
  return (int)(n < 1 ? 1 : n > most ? most : n);
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
    const int per_token = (2 * num_kv_heads) << lanes_log2;
    auto go = [&](auto kernel, int u) {
      const int64_t batch = tokens_per_batch(u, per_token);
      const int batches = batches_per_cta(nnz, batch, sms, kResident);
      return launch(kernel, dim3((unsigned)ceil_div(nnz, batch * batches)), dim3(kThreads), smem,
                    stream,
                    static_cast<const T*>(key), static_cast<const T*>(value), append_indptr,
                    static_cast<uint8_t*>(codes), static_cast<uint8_t*>(exponents), kv_indices,
                    kv_indptr, kv_last_page_len, job, batches, bad_tokens);
    };
    cudaError_t err;
    if (!vec)
      err = go(kv_quant_append_kernel<T, 1, false>, 1);
    else if (nnz <= 4 * sms)  // 100 tokens 2.5 us a launch (two a batch: 2.7), 1000 tokens 4.1 (3.8)
      err = go(kv_quant_append_kernel<T, 1, true>, 1);
    else
      err = go(kv_quant_append_kernel<T, 2, true>, 2);
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
      const int64_t batch = tokens_per_batch(u, per_token);
      const int batches = batches_per_cta(rows, batch, sms, kResident);
      return launch(kernel, dim3((unsigned)ceil_div(rows, batch * batches)), dim3(kThreads), smem,
                    stream,
                    static_cast<T*>(key), static_cast<T*>(value), out_indptr,
                    static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(exponents),
                    kv_indices, kv_indptr, kv_last_page_len, job, batches, bad_tokens);
    };
    // one round of loads a batch while that keeps every SM's threads busy once: 2300 rows 4.6 us
    // (two rounds: 5.5), 4000 rows 8.1 (7.6)
    const bool few = rows * per_token <= (int64_t)8 * kThreads * sms;
    cudaError_t err;
    if (!vec)
      err = codes_per == 16 ? go(kv_quant_read_kernel<T, 16, 1, false>, 1)
                            : go(kv_quant_read_kernel<T, 8, 1, false>, 1);
    else if (codes_per == 16)
      err = few ? go(kv_quant_read_kernel<T, 16, 1, true>, 1)
                : go(kv_quant_read_kernel<T, 16, 2, true>, 2);
    else
      err = go(kv_quant_read_kernel<T, 8, 2, true>, 2);
    if (err != cudaSuccess) return cuda_fail(err, what);
    return (int)PACE_OK;
  });
}
