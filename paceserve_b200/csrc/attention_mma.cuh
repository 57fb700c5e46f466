// Warp-level pieces of the paged-attention kernels: asynchronous copies, the
// 16 x 8 x 16 matrix instruction for both 16-bit types, unpacking of e4m3
// codes, and the joining of pieces' results.
#pragma once

#include <type_traits>

#include "attention.cuh"

namespace pace {
namespace attn {

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// 16 bytes to shared memory; zeros where `there` is false (nothing is read).
__device__ __forceinline__ void cp_async16(void* dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(dst)), "l"(src),
               "r"(there ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(smem_addr(p))
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(smem_addr(p))
               : "memory");
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Where P is fp16 it is built as 2^(s - m + kHeadroom): with a maximum that lags by
// up to 2^8 it stays below 2^16, and weights down to 2^-21 of the largest keep all
// their bits, where fp16 would else give out at 2^-14.  The sum has the same units,
// and what leaves the kernel as the maximum is m - kHeadroom.
constexpr float kHeadroom = 7.f;

// A word of four codes as two registers of two 16-bit values each, bytes 0, 2
// and bytes 1, 3: sign to the top, exponent and mantissa below it, shifted to
// the type's mantissa end.  The value is the code's times 2^-120 (bf16) or 2^-8
// (fp16).
template <int SHIFT>
__device__ __forceinline__ void spread_codes(uint32_t w, uint32_t& even, uint32_t& odd) {
  constexpr uint32_t kMag = 0x007f007fu << SHIFT;
  even = ((w << 8) & 0x80008000u) | ((w << SHIFT) & kMag);
  odd = (w & 0x80008000u) | ((w >> (8 - SHIFT)) & kMag);
}

template <typename T>
struct Mma;

template <>
struct Mma<__nv_bfloat16> {
  __device__ static __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                             uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  __device__ static __forceinline__ uint32_t pack(float x, float y) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  __device__ static __forceinline__ uint32_t pair(__nv_bfloat16 x, __nv_bfloat16 y) {
    const __nv_bfloat162 h = __halves2bfloat162(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  __device__ static __forceinline__ float2 floats(uint32_t x) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x));
  }
  __device__ static __forceinline__ uint32_t mul2(uint32_t x, uint32_t f) {
    const __nv_bfloat162 r = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&x),
                                     *reinterpret_cast<const __nv_bfloat162*>(&f));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  __device__ static __forceinline__ void unpack_codes(uint32_t w, uint32_t& even, uint32_t& odd) {
    spread_codes<4>(w, even, odd);
  }
  // Sixteen codes of a row with exponent byte `ex` as values, dimensions 0, 2, 1, 3 of each four.
  __device__ static __forceinline__ void dequantise16(const uint32_t (&w)[4], uint32_t ex,
                                                      uint32_t (&o)[8]) {
    // 2^(ex - 127 + 120) while bf16 holds it; larger rows (and NaN ones) in two steps
    const uint32_t f1 = (min(ex, 134u) + 120u) << 7, f = f1 | f1 << 16;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t a, b;
      unpack_codes(w[i], a, b);
      o[2 * i] = mul2(a, f);
      o[2 * i + 1] = mul2(b, f);
    }
    if (ex > 134u) {
      const uint32_t g1 = ex == (uint32_t)kNanExponent ? 0x7fc0u : (ex - 7u) << 7, g = g1 | g1 << 16;
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = mul2(o[i], g);
    }
  }
};

template <>
struct Mma<__half> {
  __device__ static __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                             uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  __device__ static __forceinline__ uint32_t pack(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  __device__ static __forceinline__ uint32_t pair(__half x, __half y) {
    const __half2 h = __halves2half2(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  __device__ static __forceinline__ float2 floats(uint32_t x) {
    return __half22float2(*reinterpret_cast<const __half2*>(&x));
  }
  __device__ static __forceinline__ uint32_t mul2(uint32_t x, uint32_t f) {
    const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&x),
                              *reinterpret_cast<const __half2*>(&f));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  __device__ static __forceinline__ void unpack_codes(uint32_t w, uint32_t& even, uint32_t& odd) {
    spread_codes<7>(w, even, odd);
  }
  // As above; values past fp16's range saturate.
  __device__ static __forceinline__ void dequantise16(const uint32_t (&w)[4], uint32_t ex,
                                                      uint32_t (&o)[8]) {
    uint32_t f, g;
    const float x = exponent_factor(ex);
    split_factors(x, x, f, g);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t a, b;
      unpack_codes(w[i], a, b);
      o[2 * i] = scale2(a, f, g);
      o[2 * i + 1] = scale2(b, f, g);
    }
  }
  // Two rows' factors times 2^8, as a product f * g of which fp16 holds each: g is 1 unless a
  // factor passes 2^7 (the product ends at 2^22, past which every value but a few subnormal codes
  // is outside fp16's range).  Factors below 2^-32 vanish: so do their values, in fp16.
  __device__ static __forceinline__ void split_factors(float x, float y, uint32_t& f, uint32_t& g) {
    f = pack(x != x ? x : fminf(x, 128.f) * 256.f, y != y ? y : fminf(y, 128.f) * 256.f);
    g = pack(fminf(fmaxf(x * 0.0078125f, 1.f), 32768.f), fminf(fmaxf(y * 0.0078125f, 1.f), 32768.f));
  }
  // Values past fp16's range saturate.
  __device__ static __forceinline__ uint32_t scale2(uint32_t x, uint32_t f, uint32_t g) {
    x = mul2(x, f);
    if (g != 0x3c003c00u) {
      x = mul2(x, g);
      __half2 h = *reinterpret_cast<__half2*>(&x);
      const __half2 top = __float2half2_rn(65504.f);
      h = __hmin2_nan(__hmax2_nan(h, __hneg2(top)), top);
      x = *reinterpret_cast<uint32_t*>(&h);
    }
    return x;
  }
};

// Four outputs of one row from its unnormalised sums, and the row's lse (m in
// powers of two).  A row that saw nothing (sum 0) is zero.  Returns false where a
// hidden key may have spoilt one: some are infinite or NaN, and the sum, which no
// hidden key enters, is not.
template <typename T>
__device__ __forceinline__ bool write_out(const Problem& p, int64_t tok, int head, int d,
                                          const float (&v)[4], float m, float sum) {
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  T* o = static_cast<T*>(p.out) + tok * p.out_stride + (int64_t)head * p.head_dim + d;
  T y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = Traits<T>::from_f(sum == 0.f ? 0.f : v[i] * inv);
  if ((reinterpret_cast<uintptr_t>(o) & 7) == 0) {
    *reinterpret_cast<uint2*>(o) = *reinterpret_cast<const uint2*>(y);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = y[i];
  }
  if (p.lse && d == 0)
    p.lse[tok * p.heads + head] = sum == 0.f ? -INFINITY : m * 0.6931471805599453f + logf(sum);
  return !(sum < INFINITY) ||
         fabsf(v[0] * inv) + fabsf(v[1] * inv) + fabsf(v[2] * inv) + fabsf(v[3] * inv) < INFINITY;
}

// Whether the value row of some key of [begin, end) that this row does not see
// would spoil a product with 0: an infinity or a NaN in it (of a quantised row, as
// either kernel may unpack it).  Lane by lane a key.
template <typename T, bool Q8, int D>
__device__ bool hidden_spoils(const Problem& p, int64_t tok, int head, int begin, int end) {
  const TokenInfo info = p.tokens[tok];
  const uint64_t* bits = p.tree_mask ? p.tree_mask + tok * p.tree_words : nullptr;
  const int kvh = head / (p.heads / p.kv_heads);
  const uint8_t* cache = static_cast<const uint8_t*>(p.cache);
  constexpr int kRowBytes = Q8 ? D : 2 * D;
  constexpr uint32_t kBad = Q8                                       ? 0x7f7f7f7fu
                            : std::is_same<T, __nv_bfloat16>::value ? 0x7f807f80u
                                                                    : 0x7c007c00u;
  for (int j0 = begin; j0 < end; j0 += 32) {
    const int j = j0 + (int)(threadIdx.x & 31);
    bool see = j >= info.lo && j < info.hi;
    if (bits && j >= info.hi) see = j < info.pos && tree_bit(bits, j - info.hi);
    bool bad = false;
    if (j < end && !see) {
      const int64_t page = p.kv_indices[info.page_base + page_number(p, j)];
      const int64_t row = ((page * 2 + 1) * p.page_size + page_slot(p, j)) * p.kv_heads + kvh;
      // from 2^119 on a factor may take a code past bf16's range
      if constexpr (Q8) bad = p.exponents[row] >= 127 + 119;
#pragma unroll 4
      for (int c = 0; c < kRowBytes; c += 16) {
        const uint4 x = ld_v4(cache + row * kRowBytes + c);
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          bad |= (Q8 ? __vcmpeq4(w[i] & kBad, kBad) : __vcmpeq2(w[i] & kBad, kBad)) != 0;
      }
    }
    if (__any_sync(0xffffffffu, bad)) return true;
  }
  return false;
}

// A row that came out infinite or NaN, or (`faint`) as too little of what it was
// scaled for, by attend_row; not where its own keys made it so, which NaN does to
// whole prompts (8192 such rows and heads took 500 times a finite prompt's time).
// Out of line: it is rarely needed.
template <typename T, bool Q8, int D>
__device__ __noinline__ void attend_row_again(const Problem& p, int64_t tok, int head, int begin,
                                              int end, bool faint) {
  if (faint || hidden_spoils<T, Q8, D>(p, tok, head, begin, end))
    attend_row<T, std::conditional_t<Q8, uint8_t, T>, D / 32>(p, tok, head);
}

// Redoes rows whose outputs, just written by this warp's lanes (lane u: four
// columns of row `r`), are not fine.  The whole warp calls it; lanes without a row
// pass fine = true.
template <typename T, int D, bool Q8>
__device__ __forceinline__ void redo_rows(const Problem& p, const Item& w, int kvh, int group, int r,
                                          bool fine, bool faint) {
  uint32_t bad = __ballot_sync(0xffffffffu, !fine || faint);
  const uint32_t faint_lanes = __ballot_sync(0xffffffffu, faint);
  if (bad) __syncwarp();  // their stores come before the ones below
  constexpr uint32_t kRowLanes = D / 4 >= 32 ? 0xffffffffu : (1u << (D / 4 & 31)) - 1u;
  while (bad) {
    const int first = __ffs(bad) - 1;
    const int row = __shfl_sync(0xffffffffu, r, first);
    attend_row_again<T, Q8, D>(p, w.tok0 + row / group, kvh * group + row % group, w.all_begin,
                               w.all_end, faint_lanes >> first & 1);
    bad &= ~(kRowLanes << (first / (D / 4) * (D / 4)));
  }
}

// Called by every thread of the CTA after it wrote its part of a piece's
// result: true in the CTA that arrives last of `splits`, which then sees what
// all of them wrote; the counter is zero again.
__device__ __forceinline__ bool arrive_last(int32_t* counter, int splits, bool* last) {
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    const int before = atomicAdd(counter, 1);
    *last = before == splits - 1;
    if (*last) *counter = 0;
  }
  __syncthreads();
  if (!*last) return false;
  __threadfence();
  return true;
}

template <int NT>
__device__ __forceinline__ void join_sync() {
  asm volatile("bar.sync 2, %0;" ::"n"(NT) : "memory");
}

// Joins the pieces of item w's rows and writes the output: threads 0 .. NT - 1.
// ROWS: rows of a slot; scratch: `room` floats of shared memory.  The pieces'
// weights 2^(m_k - M) are found once per row; then every thread keeps four
// columns of four units, a piece of each, in flight (one unit at a time, each
// waiting for its own loads, 32 trees took 155 us instead of 105 uncut).  A
// negative sum asks for the row to be done again.
template <typename T, int ROWS, int D, bool Q8, int NT>
__device__ __forceinline__ void join_pieces(const Problem& p, const float* partial,
                                            const float2* partial_ml, const Item& w, int kvh,
                                            int group, int rows, float* scratch, int room) {
  constexpr int V4 = D / 4, U = 4;
  const int64_t first = (int64_t)w.slot * p.kv_heads + kvh;
  const int most = min(rows, room / (2 * w.splits + 2));  // rows of a pass
  for (int r0 = 0; r0 < rows; r0 += most) {
    const int n = min(most, rows - r0);
    float *ms = scratch, *ls = ms + n * w.splits, *top = ls + n * w.splits, *total = top + n;
    for (int x = threadIdx.x; x < n * w.splits; x += NT) {
      const int k = x / n, r = x - k * n;
      const float2 ml = __ldcg(partial_ml + (first + (int64_t)k * p.kv_heads) * ROWS + r0 + r);
      ms[x] = ml.x;
      ls[x] = ml.y;
    }
    join_sync<NT>();
    for (int r = threadIdx.x; r < n; r += NT) {
      float mm = -INFINITY, sum = 0.f;
      bool redo = false;
      for (int k = 0; k < w.splits; ++k) mm = fmaxf(mm, ms[k * n + r]);
      const float b = mm == -INFINITY ? 0.f : mm;
      for (int k = 0; k < w.splits; ++k) {
        const float f = exp2_approx(ms[k * n + r] - b);
        sum += f * fabsf(ls[k * n + r]);
        redo |= ls[k * n + r] < 0.f;
        ms[k * n + r] = f;
      }
      top[r] = mm;
      total[r] = redo ? -sum : sum;
    }
    join_sync<NT>();
    // whole warps stay in the loop, for redo_rows
    for (int u0 = threadIdx.x; (u0 & ~31) < n * V4; u0 += U * NT) {
      float v[U][4];
#pragma unroll
      for (int i = 0; i < U; ++i) v[i][0] = v[i][1] = v[i][2] = v[i][3] = 0.f;
#pragma unroll 2
      for (int k = 0; k < w.splits; ++k) {
        const float* piece = partial + ((first + (int64_t)k * p.kv_heads) * ROWS + r0) * D;
#pragma unroll
        for (int i = 0; i < U; ++i) {
          const int u = u0 + i * NT;
          if (u < n * V4) {
            const float4 x = __ldcg(reinterpret_cast<const float4*>(piece) + u);
            const float f = ms[k * n + u / V4];
            v[i][0] += f * x.x;
            v[i][1] += f * x.y;
            v[i][2] += f * x.z;
            v[i][3] += f * x.w;
          }
        }
      }
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int u = u0 + i * NT;
        if ((u & ~31) >= n * V4) break;
        const int r = u / V4;
        bool fine = true, faint = false;
        if (u < n * V4) {
          fine = write_out<T>(p, w.tok0 + (r0 + r) / group, kvh * group + (r0 + r) % group,
                              (u - r * V4) * 4, v[i], top[r], fabsf(total[r])) ||
                 !w.mixed;
          faint = Q8 && total[r] < 0.f;
        }
        if (w.mixed || Q8) redo_rows<T, D, Q8>(p, w, kvh, group, r0 + r, fine, faint);
      }
    }
    join_sync<NT>();
  }
}

// The two tensor-core kernels' launchers.
int run_tile_rows(const Problem& p, int64_t num_pages, const Item* items, int num_items, float* partial, float2* ml,
                  int32_t* counters, int32_t* fault, bool bf16, int device, cudaStream_t stream,
                  const char* what);
int run_few_rows(const Problem& p, int max_rows, const Item* items, int num_items, float* partial,
                 float2* ml, int32_t* counters, bool beside, bool bf16, int device,
                 cudaStream_t stream, const char* what);

}  // namespace attn
}  // namespace pace
