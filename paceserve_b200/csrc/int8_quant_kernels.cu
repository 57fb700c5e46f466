// Rows as 8-bit integers with a scale each, for sm_100a: of a tensor, of an
// RMSNorm (with the residual added first), or of SiLU-and-mul.
//
//   scale_t = max(max_k |y_tk| / 127, 2^-126),   code_tk = rint(y_tk / scale_t)
//   y = x;   y = r * rsqrt(mean r^2 + eps) * w with r = (T)(x + residual);   y = silu(g) * u
//
// y is fp32 and is never rounded to T: the code's half step is the one rounding
// (and r's, since r is the residual stream that the next layer reads).  A row
// with an infinity or a NaN in y has no scale: its scale is NaN and its codes 0,
// so that all that is computed from it is NaN.
//
// The quotient is rounded as IEEE division gives it, without a division for
// each element: y * (1 / scale) is off by less than 2^-15 at 127, so only where
// it falls within 1e-4 of a half step can the nearest integer be another, and
// there (four elements in 1250 times) the division is done.
//
// Memory bounds it: a row is read once with 16-byte vectors, held in registers
// over the one or two reductions, and stored as 8-byte groups of codes.  Between
// its loads and its stores a CTA has nothing under way, so each also asks for the
// row a CTA of the next wave will read, into L2 (8192 rows of SiLU-and-mul, 14336
// codes: 104 us, 5.6 TB/s, against 110; 1999 rows 29 against 30.5).
#include "f32x2.cuh"

namespace pace {
namespace {

enum Source { kRows, kNorm, kAddNorm, kSilu };
constexpr int kMaxThreads = 512, kWideThreads = 1024;  // wide: rows that need more
constexpr float kLeastScale = 1.17549435e-38f;  // 2^-126

struct QuantJob {
  int8_t* codes;
  float* scales;
  const void* x;
  void* residual;      // kAddNorm
  const void* weight;  // kNorm, kAddNorm
  float eps;
  int width;  // codes per row
  int64_t x_stride, residual_stride, codes_stride;
  int ahead;  // rows, of the asking ahead
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  return v;
}

// Sum over the CTA, the same for every thread.
__device__ __forceinline__ float block_sum(float v, float* red) {
  v = warp_sum(v);
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  if (lane == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  return warp_sum(lane < warps ? red[lane] : 0.f);
}

// Largest magnitude over the CTA, of the threads' own; NaN if any is.
__device__ __forceinline__ float block_max(float v, uint32_t* red) {
  // as bit patterns, whose order is that of magnitudes, with infinity and NaN above all
  uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(v) & 0x7fffffffu);
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  if (lane == 0) red[threadIdx.x >> 5] = bits;
  __syncthreads();
  bits = __reduce_max_sync(0xffffffffu, lane < warps ? red[lane] : 0u);
  return __uint_as_float(bits);
}

// The larger magnitude, NaN if either is.
__device__ __forceinline__ float larger(float top, float y) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(top), "f"(fabsf(y)));
  return r;
}

// silu(g) * u of two elements.  16-bit inputs take the approximate exponential and
// reciprocal, float32 the library's.  The approximate exponential's argument is
// rounded, which leaves an error that goes with |g|: at most (4 |g| + 16) 2^-24 of the
// value, at |g| = 100 a 150th of the code's half step.
template <typename T>
__device__ __forceinline__ void silu_mul2(float* g, const float* u) {
  if constexpr (sizeof(T) == 2) {
    float a, b, c, d;
    apart(mul2(two(g[0], g[1]), two(-1.44269504f, -1.44269504f)), a, b);
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(c) : "f"(a));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(d) : "f"(b));
    apart(add2(two(c, d), two(1.f, 1.f)), a, b);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(c) : "f"(a));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(d) : "f"(b));
    apart(mul2(mul2(two(g[0], g[1]), two(c, d)), two(u[0], u[1])), g[0], g[1]);
  } else {
    g[0] = g[0] / (1.f + expf(-g[0])) * u[0];
    g[1] = g[1] / (1.f + expf(-g[1])) * u[1];
  }
}

struct RowScale {
  float scale, inverse;
  bool finite;
  __device__ __forceinline__ explicit RowScale(float top) {
    finite = top <= 3.402823466e38f;
    scale = finite ? fmaxf(__fdiv_rn(top, 127.f), kLeastScale) : __uint_as_float(0x7fc00000u);
    inverse = __fdiv_rn(1.f, scale);
  }
  // Four codes, the first in the low byte.
  __device__ __forceinline__ uint32_t four(const float* y) const {
    constexpr float kInteger = 12582912.f;  // 1.5 * 2^23: adding it leaves an integer in the low bits
    const uint64_t inv = two(inverse, inverse), up = two(kInteger, kInteger), minus = two(-1.f, -1.f);
    float r[4], off[4];
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
      const uint64_t v = two(y[e], y[e + 1]), s = fma2(v, inv, up);
      apart(s, r[e], r[e + 1]);
      apart(fma2(v, inv, fma2(s, minus, up)), off[e], off[e + 1]);  // from the integer
    }
    const float most = fmaxf(fmaxf(fabsf(off[0]), fabsf(off[1])), fmaxf(fabsf(off[2]), fabsf(off[3])));
    if (most > 0.4999f) {  // near a half step the quotient itself decides
#pragma unroll
      for (int e = 0; e < 4; ++e) r[e] = __fdiv_rn(y[e], scale) + kInteger;
    }
    if (!finite) return 0u;
    const uint32_t lo = __byte_perm(__float_as_uint(r[0]), __float_as_uint(r[1]), 0x0040);
    const uint32_t hi = __byte_perm(__float_as_uint(r[2]), __float_as_uint(r[3]), 0x0040);
    return __byte_perm(lo, hi, 0x5410);
  }
  __device__ __forceinline__ int8_t one(float y) const {
    const float v[4] = {y, 0.f, 0.f, 0.f};
    return (int8_t)four(v);
  }
};

template <typename T, int SRC, int NV, int THREADS = kMaxThreads>
__global__ void __launch_bounds__(THREADS) quantise_vec_kernel(const QuantJob job) {
  using Tr = Traits<T>;
  constexpr int V = Tr::kVec;
  __shared__ float red_sum[32];
  __shared__ uint32_t red_max[32];
  const int64_t row = blockIdx.x;
  const int nvec = job.width / V;
  const T* xr = static_cast<const T*>(job.x) + row * job.x_stride;
  T* rr = SRC == kAddNorm ? static_cast<T*>(job.residual) + row * job.residual_stride : nullptr;
  const T* weight = static_cast<const T*>(job.weight);
  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    const int64_t bytes = (int64_t)job.width * sizeof(T), read = SRC == kSilu ? 2 * bytes : bytes;
    prefetch_l2(xr, read);
    if (SRC == kAddNorm) prefetch_l2(rr, bytes);
    if (row + job.ahead < gridDim.x) {
      prefetch_l2(xr + job.ahead * job.x_stride, read);
      if (SRC == kAddNorm) prefetch_l2(rr + job.ahead * job.residual_stride, bytes);
    }
    if ((SRC == kNorm || SRC == kAddNorm) && row < 4) prefetch_l2(weight, bytes);
  }
  pdl_wait();
  uint4 a[NV], b[NV], w[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = threadIdx.x + j * blockDim.x;
    if (c < nvec) {
      a[j] = ld_nc_v4(xr + (int64_t)c * V);
      if (SRC == kSilu) b[j] = ld_nc_v4(xr + job.width + (int64_t)c * V);
      if (SRC == kAddNorm) b[j] = ld_v4(rr + (int64_t)c * V);
      if (SRC == kNorm || SRC == kAddNorm) w[j] = __ldg(reinterpret_cast<const uint4*>(weight) + c);
    }
  }
  float y[NV][V];
  uint64_t ss = 0;
  float top = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = threadIdx.x + j * blockDim.x;
    if (c < nvec) {
      Tr::unpack(a[j], y[j]);
      if constexpr (SRC == kSilu || SRC == kAddNorm) {
        float z[V];
        Tr::unpack(b[j], z);
#pragma unroll
        for (int e = 0; e < V; e += 2) {
          if constexpr (SRC == kSilu) {
            silu_mul2<T>(y[j] + e, z + e);
          } else {
            y[j][e] = Tr::round(y[j][e] + z[e]);
            y[j][e + 1] = Tr::round(y[j][e + 1] + z[e + 1]);
          }
        }
        if (SRC == kAddNorm) st_v4(rr + (int64_t)c * V, Tr::pack(y[j]));
      }
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        const uint64_t v = two(y[j][e], y[j][e + 1]);
        if (SRC == kNorm || SRC == kAddNorm)
          ss = fma2(v, v, ss);
        else
          top = larger(larger(top, y[j][e]), y[j][e + 1]);
      }
    }
  }
  if constexpr (SRC == kNorm || SRC == kAddNorm) {
    float lo, hi;
    apart(ss, lo, hi);
    const float inv = rsqrtf(block_sum(lo + hi, red_sum) / (float)job.width + job.eps);
    const uint64_t inv2 = two(inv, inv);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = threadIdx.x + j * blockDim.x;
      if (c < nvec) {
        float wf[V];
        Tr::unpack(w[j], wf);
#pragma unroll
        for (int e = 0; e < V; e += 2) {
          apart(mul2(mul2(two(y[j][e], y[j][e + 1]), inv2), two(wf[e], wf[e + 1])), y[j][e],
                y[j][e + 1]);
          top = larger(larger(top, y[j][e]), y[j][e + 1]);
        }
      }
    }
  }
  const RowScale s(block_max(top, red_max));
  if (threadIdx.x == 0) job.scales[row] = s.scale;
  int8_t* codes = job.codes + row * job.codes_stride;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = threadIdx.x + j * blockDim.x;
    if (c < nvec) {
      if constexpr (SRC == kRows && sizeof(T) == 2) {
        // the row was held as it came, half the registers: 14336 wide, 2000 rows 24.9 us with fp32
        asm volatile("" : "+r"(a[j].x), "+r"(a[j].y), "+r"(a[j].z), "+r"(a[j].w));
        Tr::unpack(a[j], y[j]);
      }
      uint32_t word[V / 4];
#pragma unroll
      for (int i = 0; i < V / 4; ++i) word[i] = s.four(y[j] + 4 * i);
      if constexpr (V == 8)
        *reinterpret_cast<uint2*>(codes + (int64_t)c * V) = make_uint2(word[0], word[1]);
      else
        *reinterpret_cast<uint32_t*>(codes + (int64_t)c * V) = word[0];
    }
  }
}

// Any width, stride and alignment: a thread's elements are computed anew in
// each pass, from what it read (and, with a residual, wrote) itself.
template <typename T, int SRC>
__global__ void __launch_bounds__(256) quantise_scalar_kernel(const QuantJob job) {
  using Tr = Traits<T>;
  __shared__ float red_sum[32];
  __shared__ uint32_t red_max[32];
  const int64_t row = blockIdx.x;
  const T* xr = static_cast<const T*>(job.x) + row * job.x_stride;
  T* rr = SRC == kAddNorm ? static_cast<T*>(job.residual) + row * job.residual_stride : nullptr;
  const T* weight = static_cast<const T*>(job.weight);
  pdl_launch_dependents();
  pdl_wait();
  float inv = 1.f;
  if constexpr (SRC == kNorm || SRC == kAddNorm) {
    float ss = 0.f;
    for (int i = threadIdx.x; i < job.width; i += blockDim.x) {
      float v = Tr::to_f(xr[i]);
      if (SRC == kAddNorm) {
        v = Tr::round(v + Tr::to_f(rr[i]));
        rr[i] = Tr::from_f(v);
      }
      ss += v * v;
    }
    inv = rsqrtf(block_sum(ss, red_sum) / (float)job.width + job.eps);
  }
  auto value = [&](int i) -> float {
    if constexpr (SRC == kSilu) {
      float g[2] = {Tr::to_f(xr[i]), 0.f};
      const float u[2] = {Tr::to_f(xr[job.width + i]), 0.f};
      silu_mul2<T>(g, u);
      return g[0];
    }
    if constexpr (SRC == kNorm) return Tr::to_f(xr[i]) * inv * Tr::to_f(weight[i]);
    if constexpr (SRC == kAddNorm) return Tr::to_f(rr[i]) * inv * Tr::to_f(weight[i]);
    return Tr::to_f(xr[i]);
  };
  float top = 0.f;
  for (int i = threadIdx.x; i < job.width; i += blockDim.x) top = larger(top, value(i));
  const RowScale s(block_max(top, red_max));
  if (threadIdx.x == 0) job.scales[row] = s.scale;
  int8_t* codes = job.codes + row * job.codes_stride;
  for (int i = threadIdx.x; i < job.width; i += blockDim.x) codes[i] = s.one(value(i));
}

// Threads a row, at most: many rows do best with several vectors a thread (4096
// wide, norm with residual, us, 128 / 256 / 512 threads: 512 rows 6.4, 5.7, 4.4;
// 2048 rows 12.3, 12.2, 13.7; 8192 rows 39, 41, 49), few rows, a CTA an SM, with the
// shortest chain (SiLU-and-mul of 14336 codes, 256 / 512 / 1024 threads: 64 rows
// 4.8, 4.7, 3.3; 256 rows 5.7, 5.7, 6.4).
inline int most_threads(int64_t rows, int sms) {
  return rows > 4096 ? 128 : rows > 1024 ? 256 : rows > sms ? kMaxThreads : kWideThreads;
}

template <typename T, int SRC>
int launch_quantise(QuantJob job, int64_t rows, int device, cudaStream_t stream, const char* name) {
  constexpr int V = Traits<T>::kVec;
  const int64_t nvec = job.width / V;
  bool vec = job.width % V == 0 && job.x_stride % V == 0 && job.codes_stride % V == 0 &&
             aligned16(job.x) && (reinterpret_cast<uintptr_t>(job.codes) & (V - 1)) == 0 &&
             nvec <= 4 * kWideThreads;
  if (SRC == kNorm || SRC == kAddNorm) vec = vec && aligned16(job.weight);
  if (SRC == kAddNorm) vec = vec && job.residual_stride % V == 0 && aligned16(job.residual);
  const dim3 grid((unsigned)rows);
  cudaError_t err;
  if (vec) {
    const int sms = sm_count(device);
    job.ahead = sms;
    int nv = 1;
    while (nv < 4 && ceil_div(nvec, nv) > most_threads(rows, sms)) nv *= 2;
    const dim3 threads((unsigned)(ceil_div(ceil_div(nvec, nv), 32) * 32));
    // more than 512 threads leave a thread 64 registers (2048 rows of SiLU-and-mul, 18432 codes: 35.6 us;
    // element by element 165)
    auto go = [&](auto few, auto wide) {
      return launch(threads.x > kMaxThreads ? wide : few, grid, threads, 0, stream, job);
    };
    err = nv == 1   ? go(quantise_vec_kernel<T, SRC, 1>, quantise_vec_kernel<T, SRC, 1, kWideThreads>)
          : nv == 2 ? go(quantise_vec_kernel<T, SRC, 2>, quantise_vec_kernel<T, SRC, 2, kWideThreads>)
                    : go(quantise_vec_kernel<T, SRC, 4>, quantise_vec_kernel<T, SRC, 4, kWideThreads>);
  } else {
    err = launch(quantise_scalar_kernel<T, SRC>, grid, dim3(256), 0, stream, job);
  }
  return err == cudaSuccess ? PACE_OK : cuda_fail(err, name);
}

// What the entry points have in common: shapes, pointers, the number types.
template <typename F>
int checked(const QuantJob& job, int64_t rows, int64_t width, int64_t inputs, bool pointers,
            const char* name, F run) {
  if (rows < 0 || rows > INT32_MAX || width <= 0 || width > (1 << 30))
    return fail(PACE_ERR_INVALID_ARGUMENT, "%s: bad shape [%lld, %lld]", name, (long long)rows,
                (long long)width);
  if (job.x_stride < inputs * width || job.codes_stride < width)
    return fail(PACE_ERR_INVALID_ARGUMENT, "%s: row stride smaller than the row", name);
  if (rows == 0) return PACE_OK;
  if (!job.codes || !job.scales || !job.x || !pointers)
    return fail(PACE_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
  return run();
}

}  // namespace
}  // namespace pace

extern "C" int pace_quantise_rows(int8_t* codes, float* scales, const void* input, int64_t rows,
                                  int64_t width, int64_t input_row_stride,
                                  int64_t codes_row_stride, int dtype, cudaStream_t stream) {
  using namespace pace;
  const QuantJob job{codes, scales,     input,            nullptr, nullptr,
                     0.f,   (int)width, input_row_stride, 0,       codes_row_stride};
  return checked(job, rows, width, 1, true, "quantise_rows", [&] {
    StreamDeviceGuard guard(stream);
    return PACE_DISPATCH_FLOAT(dtype, "quantise_rows", [&] {
      return launch_quantise<scalar_t, kRows>(job, rows, guard.device(), stream, "quantise_rows");
    });
  });
}

extern "C" int pace_rms_norm_quantise(int8_t* codes, float* scales, const void* input,
                                      void* residual, const void* weight, float epsilon,
                                      int64_t num_tokens, int64_t hidden_size,
                                      int64_t input_row_stride, int64_t residual_row_stride,
                                      int64_t codes_row_stride, int dtype, cudaStream_t stream) {
  using namespace pace;
  const QuantJob job{codes,
                     scales,
                     input,
                     residual,
                     weight,
                     epsilon,
                     (int)hidden_size,
                     input_row_stride,
                     residual_row_stride,
                     codes_row_stride};
  if (residual && residual_row_stride < hidden_size)
    return fail(PACE_ERR_INVALID_ARGUMENT, "rms_norm_quantise: row stride smaller than the row");
  return checked(job, num_tokens, hidden_size, 1, weight != nullptr, "rms_norm_quantise", [&] {
    StreamDeviceGuard guard(stream);
    return PACE_DISPATCH_FLOAT(dtype, "rms_norm_quantise", [&] {
      return residual ? launch_quantise<scalar_t, kAddNorm>(job, num_tokens, guard.device(), stream,
                                                            "rms_norm_quantise")
                      : launch_quantise<scalar_t, kNorm>(job, num_tokens, guard.device(), stream,
                                                         "rms_norm_quantise");
    });
  });
}

extern "C" int pace_silu_and_mul_quantise(int8_t* codes, float* scales, const void* input,
                                          int64_t num_tokens, int64_t d, int64_t input_row_stride,
                                          int64_t codes_row_stride, int dtype,
                                          cudaStream_t stream) {
  using namespace pace;
  const QuantJob job{codes, scales, input,            nullptr, nullptr,
                     0.f,   (int)d, input_row_stride, 0,       codes_row_stride};
  return checked(job, num_tokens, d, 2, true, "silu_and_mul_quantise", [&] {
    StreamDeviceGuard guard(stream);
    return PACE_DISPATCH_FLOAT(dtype, "silu_and_mul_quantise", [&] {
      return launch_quantise<scalar_t, kSilu>(job, num_tokens, guard.device(), stream,
                                              "silu_and_mul_quantise");
    });
  });
}
