// RMSNorm of every query and key head and the rotary embedding in one pass, in
// place or with the keys and values written to their slots of the paged cache,
// for sm_100a.
//
//   y = x * rsqrt(mean_d x^2 + eps) * w   over one head's dimensions, w of the queries or the keys
//   NeoX:  (y_i, y_{i + rot/2}),  GPT-J: (y_2i, y_{2i+1})   for i < rot / 2, rotated by the
//   angle whose cosine and sine the position's row of the cache holds; the rest stays y.
//
// All in fp32, rounded once.  It is bound by memory: q, k (and v) are read once
// and written once, where norm, rotation and append as separate passes read and
// write the keys three times.  Rotation and norm keep the layout and the
// position rule of rotary_embedding (a token whose position is outside the
// table stays as it is); the cache's layout is that of append_paged_kv_cache
// (flashinfer_attention_wrapper.py:53-73), addressed by slot = page * page_size
// + place in the page.
//
// A head belongs to G neighbouring lanes, each with two 16-byte vectors: a
// rotation's two halves (NeoX) or 2 x 8 neighbours (GPT-J), so that rotation is
// in the thread and the norm is log2(G) shuffles.  Tokens and heads are dealt to
// CTAs as one flat range, so few heads or narrow ones fill a CTA as well.
#include "common.cuh"

namespace pace {
namespace {

struct HeadJob {
  const int64_t* positions;
  void *query, *key;
  const void* value;  // APPEND
  const void *q_weight, *k_weight;
  const void* cos_sin;
  void* cache;           // APPEND
  const int64_t* slots;  // APPEND
  int32_t* bad;
  float eps;
  int num_tokens, heads, kv_heads, head_size, rot_dim;
  int page_size, page_shift;  // page_shift: log2, or -1
  int64_t q_stride, k_stride, v_stride, max_position, num_slots;
};

// N consecutive entries of the cos/sin table or a weight as floats.
template <typename C, int N>
__device__ __forceinline__ void load_floats(const C* p, float* out) {
  if constexpr (sizeof(C) == 4) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const float4 v = __ldg(reinterpret_cast<const float4*>(p) + i);
      out[4 * i] = v.x;
      out[4 * i + 1] = v.y;
      out[4 * i + 2] = v.z;
      out[4 * i + 3] = v.w;
    }
  } else {
    Traits<C>::unpack(__ldg(reinterpret_cast<const uint4*>(p)), out);
  }
}

__device__ __forceinline__ void prefetch_line(const void* p) {
  asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
}

// Where the cache holds K (0) or V (1) of a slot.
__device__ __forceinline__ int64_t cache_row(const HeadJob& j, int64_t slot, int kind) {
  int64_t page;
  int at;
  if (j.page_shift >= 0) {
    page = slot >> j.page_shift;
    at = (int)slot & (j.page_size - 1);
  } else {
    page = slot / j.page_size;
    at = (int)(slot - page * j.page_size);
  }
  return (page * 2 + kind) * j.page_size + at;
}

// Whether a token's keys and values go to the cache.  Slot -1 (a padded token)
// is passed over in silence, any other that is no slot is counted, as is a
// token with a slot but no position.
__device__ __forceinline__ bool goes_to_cache(const HeadJob& j, int64_t slot, bool placed,
                                              bool counts) {
  const bool good = slot >= 0 && slot < j.num_slots && placed;
  if (!good && counts && slot != -1 && j.bad) atomicAdd(j.bad, 1);
  return good;
}

// G: lanes of a head.  Head numbers: queries, keys, then (APPEND) values.
template <typename T, typename C, bool NEOX, bool APPEND, int G>
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(const HeadJob j) {
  using Tr = Traits<T>;
  constexpr int V = Tr::kVec;
  const int heads = j.heads + (APPEND ? 2 : 1) * j.kv_heads;
  const int lanes = heads * G;  // of a token
  const int64_t first = (int64_t)blockIdx.x * blockDim.x;
  const int64_t tok0 = first / lanes;
  const int at = (int)(first - tok0 * lanes) + (int)threadIdx.x;
  const int more = at / lanes;
  const int64_t tok = tok0 + more;
  const int head = (at - more * lanes) / G;
  const int l = threadIdx.x % G;
  const int units = j.head_size / (2 * V), turns = j.rot_dim / (2 * V);
  const bool live = tok < j.num_tokens && l < units;
  const bool is_q = head < j.heads, is_v = APPEND && head >= j.heads + j.kv_heads;
  const int h = is_q ? head : is_v ? head - j.heads - j.kv_heads : head - j.heads;
  // this lane's two vectors
  const bool turn = l < turns;
  int d0, d1;
  if (NEOX && turn) {
    d0 = l * V;
    d1 = j.rot_dim / 2 + d0;
  } else {
    d0 = l * 2 * V;
    d1 = d0 + V;
  }
  T* row = is_q   ? static_cast<T*>(j.query) + tok * j.q_stride
           : is_v ? const_cast<T*>(static_cast<const T*>(j.value)) + tok * j.v_stride
                  : static_cast<T*>(j.key) + tok * j.k_stride;
  row += (int64_t)h * j.head_size;
  pdl_launch_dependents();
  if (live) {
    prefetch_line(row + d0);
    prefetch_line(row + d1);
  }
  pdl_wait();
  uint4 xv = make_uint4(0, 0, 0, 0), yv = xv;
  int64_t pos = -1, slot = -1;
  if (live) {
    xv = ld_v4(row + d0);
    yv = ld_v4(row + d1);
    pos = j.positions[tok];
    if (APPEND && !is_q) slot = j.slots[tok];
  }
  const bool placed = pos >= 0 && pos < j.max_position;
  T* dst = row;
  bool store = live && placed;
  if (APPEND && !is_q && live) {
    store = goes_to_cache(j, slot, placed, l == 0 && head == j.heads);
    if (store)
      dst = static_cast<T*>(j.cache) +
            (cache_row(j, slot, is_v) * j.kv_heads + h) * (int64_t)j.head_size;
  }
  float x[V], y[V], c[V], s[V];
  Tr::unpack(xv, x);
  Tr::unpack(yv, y);
  if (turn && store && !is_v) {
    const C* table = static_cast<const C*>(j.cos_sin) + pos * j.rot_dim + l * V;
    load_floats<C, V>(table, c);
    load_floats<C, V>(table + j.rot_dim / 2, s);
  }
  float ss = 0.f;
#pragma unroll
  for (int e = 0; e < V; ++e) ss += x[e] * x[e] + y[e] * y[e];
#pragma unroll
  for (int m = 1; m < G; m <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
  if (!store) return;
  if (!is_v) {
    const float inv = rsqrtf(ss / (float)j.head_size + j.eps);
    const T* weight = static_cast<const T*>(is_q ? j.q_weight : j.k_weight);
    float wx[V], wy[V];
    load_floats<T, V>(weight + d0, wx);
    load_floats<T, V>(weight + d1, wy);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      x[e] = x[e] * inv * wx[e];
      y[e] = y[e] * inv * wy[e];
    }
    if (turn) {
      if constexpr (NEOX) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float a = x[e], b = y[e];
          x[e] = a * c[e] - b * s[e];
          y[e] = b * c[e] + a * s[e];
        }
      } else {
        // pairs (2i, 2i + 1): the first vector's, then the second's
#pragma unroll
        for (int e = 0; e < V; e += 2) {
          const float a = x[e], b = x[e + 1], f = y[e], g = y[e + 1];
          x[e] = a * c[e / 2] - b * s[e / 2];
          x[e + 1] = b * c[e / 2] + a * s[e / 2];
          y[e] = f * c[V / 2 + e / 2] - g * s[V / 2 + e / 2];
          y[e + 1] = g * c[V / 2 + e / 2] + f * s[V / 2 + e / 2];
        }
      }
    }
    xv = Tr::pack(x);
    yv = Tr::pack(y);
  }
  st_v4(dst + d0, xv);
  st_v4(dst + d1, yv);
}

// Any head size, stride and alignment: a warp per head; a lane reads, and then
// writes, the same rotation pairs and the same dimensions past them.
template <typename T, typename C, bool NEOX, bool APPEND>
__global__ void __launch_bounds__(128) qk_norm_rope_scalar_kernel(const HeadJob j) {
  using Tr = Traits<T>;
  const int heads = j.heads + (APPEND ? 2 : 1) * j.kv_heads;
  const int lane = threadIdx.x & 31;
  const int64_t tok = blockIdx.x;
  pdl_launch_dependents();
  pdl_wait();
  const int64_t pos = j.positions[tok];
  const bool placed = pos >= 0 && pos < j.max_position;
  const int half = j.rot_dim / 2;
  for (int head = threadIdx.x >> 5; head < heads; head += blockDim.x >> 5) {
    const bool is_q = head < j.heads, is_v = APPEND && head >= j.heads + j.kv_heads;
    const int h = is_q ? head : is_v ? head - j.heads - j.kv_heads : head - j.heads;
    const T* row = is_q   ? static_cast<const T*>(j.query) + tok * j.q_stride
                   : is_v ? static_cast<const T*>(j.value) + tok * j.v_stride
                          : static_cast<const T*>(j.key) + tok * j.k_stride;
    row += (int64_t)h * j.head_size;
    T* dst = const_cast<T*>(row);
    if (APPEND && !is_q) {
      const int64_t slot = j.slots[tok];
      if (!goes_to_cache(j, slot, placed, lane == 0 && head == j.heads)) continue;
      dst = static_cast<T*>(j.cache) +
            (cache_row(j, slot, is_v) * j.kv_heads + h) * (int64_t)j.head_size;
    } else if (!placed) {
      continue;
    }
    if (is_v) {
      for (int d = lane; d < j.head_size; d += 32) dst[d] = row[d];
      continue;
    }
    float ss = 0.f;
    for (int d = lane; d < j.head_size; d += 32) {
      const float v = Tr::to_f(row[d]);
      ss += v * v;
    }
    for (int m = 16; m > 0; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
    const float inv = rsqrtf(ss / (float)j.head_size + j.eps);
    const T* weight = static_cast<const T*>(is_q ? j.q_weight : j.k_weight);
    const C* table = static_cast<const C*>(j.cos_sin) + pos * j.rot_dim;
    for (int i = lane; i < half; i += 32) {
      const int d0 = NEOX ? i : 2 * i, d1 = NEOX ? half + i : 2 * i + 1;
      const float a = Tr::to_f(row[d0]) * inv * Tr::to_f(weight[d0]);
      const float b = Tr::to_f(row[d1]) * inv * Tr::to_f(weight[d1]);
      const float c = Traits<C>::to_f(table[i]), s = Traits<C>::to_f(table[half + i]);
      dst[d0] = Tr::from_f(a * c - b * s);
      dst[d1] = Tr::from_f(b * c + a * s);
    }
    for (int d = j.rot_dim + lane; d < j.head_size; d += 32)
      dst[d] = Tr::from_f(Tr::to_f(row[d]) * inv * Tr::to_f(weight[d]));
  }
}

template <typename T, typename C, bool NEOX, bool APPEND>
int launch_heads(const HeadJob& j, cudaStream_t stream, const char* name) {
  constexpr int V = Traits<T>::kVec;
  const int heads = j.heads + (APPEND ? 2 : 1) * j.kv_heads;
  bool vec = j.head_size % (2 * V) == 0 && j.rot_dim % (2 * V) == 0 && j.head_size <= 64 * V &&
             aligned16(j.q_weight) && aligned16(j.k_weight) && aligned16(j.cos_sin);
  if (j.heads > 0) vec = vec && j.q_stride % V == 0 && aligned16(j.query);
  if (j.kv_heads > 0) vec = vec && j.k_stride % V == 0 && aligned16(j.key);
  if (APPEND) vec = vec && j.v_stride % V == 0 && aligned16(j.value) && aligned16(j.cache);
  cudaError_t err;
  if (vec) {
    const int units = j.head_size / (2 * V);
    int g = 1;
    while (g < units) g *= 2;
    constexpr int kThreads = 256;
    const int64_t ctas = ceil_div((int64_t)j.num_tokens * heads * g, kThreads);
    if (ctas > INT32_MAX) return fail(PACE_ERR_TOO_LARGE, "%s: too many heads", name);
    auto go = [&](auto kernel) {
      return launch(kernel, dim3((unsigned)ctas), dim3(kThreads), 0, stream, j);
    };
    switch (g) {
      case 1: err = go(qk_norm_rope_kernel<T, C, NEOX, APPEND, 1>); break;
      case 2: err = go(qk_norm_rope_kernel<T, C, NEOX, APPEND, 2>); break;
      case 4: err = go(qk_norm_rope_kernel<T, C, NEOX, APPEND, 4>); break;
      case 8: err = go(qk_norm_rope_kernel<T, C, NEOX, APPEND, 8>); break;
      case 16: err = go(qk_norm_rope_kernel<T, C, NEOX, APPEND, 16>); break;
      default: err = go(qk_norm_rope_kernel<T, C, NEOX, APPEND, 32>); break;
    }
  } else {
    err = launch(qk_norm_rope_scalar_kernel<T, C, NEOX, APPEND>, dim3((unsigned)j.num_tokens),
                 dim3(128), 0, stream, j);
  }
  return err == cudaSuccess ? PACE_OK : cuda_fail(err, name);
}

template <bool APPEND>
int run_heads(const HeadJob& j, int64_t num_tokens, int cache_dtype, bool neox, int dtype,
              cudaStream_t stream, const char* name) {
  if (num_tokens < 0 || num_tokens > INT32_MAX || j.heads < 0 || j.kv_heads < 0 ||
      j.head_size <= 0 || (int64_t)(j.heads + 2 * (int64_t)j.kv_heads) * j.head_size > INT32_MAX)
    return fail(PACE_ERR_INVALID_ARGUMENT, "%s: bad shape", name);
  if (j.rot_dim <= 0 || j.rot_dim % 2 != 0 || j.rot_dim > j.head_size)
    return fail(PACE_ERR_INVALID_ARGUMENT, "%s: rot_dim %d must be even and in (0, head_size=%d]",
                name, j.rot_dim, j.head_size);
  if (j.max_position <= 0)
    return fail(PACE_ERR_INVALID_ARGUMENT, "%s: empty cos_sin_cache", name);
  const int64_t kv_row = (int64_t)j.kv_heads * j.head_size;
  if (j.q_stride < (int64_t)j.heads * j.head_size || (j.kv_heads > 0 && j.k_stride < kv_row) ||
      (APPEND && j.v_stride < kv_row))
    return fail(PACE_ERR_INVALID_ARGUMENT, "%s: row stride smaller than the row", name);
  if (APPEND && (j.kv_heads == 0 || j.page_size <= 0 || j.num_slots < 0))
    return fail(PACE_ERR_INVALID_ARGUMENT, "%s: bad cache shape", name);
  if (num_tokens == 0 || j.heads + j.kv_heads == 0) return PACE_OK;
  if (!j.positions || !j.cos_sin || !j.q_weight || !j.k_weight || (j.heads > 0 && !j.query) ||
      (j.kv_heads > 0 && !j.key) ||
      (APPEND && (!j.value || !j.slots || (!j.cache && j.num_slots > 0))))
    return fail(PACE_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
  StreamDeviceGuard guard(stream);
  return PACE_DISPATCH_FLOAT(dtype, name, [&] {
    if (cache_dtype == PACE_F32)
      return neox ? launch_heads<scalar_t, float, true, APPEND>(j, stream, name)
                  : launch_heads<scalar_t, float, false, APPEND>(j, stream, name);
    if (cache_dtype == dtype)
      return neox ? launch_heads<scalar_t, scalar_t, true, APPEND>(j, stream, name)
                  : launch_heads<scalar_t, scalar_t, false, APPEND>(j, stream, name);
    return fail(PACE_ERR_UNSUPPORTED_DTYPE,
                "%s: cos_sin_cache dtype %d must be float32 or the q/k dtype %d", name,
                cache_dtype, dtype);
  });
}

}  // namespace
}  // namespace pace

extern "C" int pace_qk_norm_rotary_embedding(
    const int64_t* positions, void* query, void* key, const void* q_weight, const void* k_weight,
    float epsilon, int64_t num_tokens, int num_heads, int num_kv_heads, int head_size,
    int64_t query_row_stride, int64_t key_row_stride, const void* cos_sin_cache, int cache_dtype,
    int rot_dim, int64_t max_position, int is_neox, int dtype, cudaStream_t stream) {
  pace::HeadJob j = {};
  j.positions = positions;
  j.query = query;
  j.key = key;
  j.q_weight = q_weight;
  j.k_weight = k_weight;
  j.cos_sin = cos_sin_cache;
  j.eps = epsilon;
  j.num_tokens = (int)num_tokens;
  j.heads = num_heads;
  j.kv_heads = num_kv_heads;
  j.head_size = head_size;
  j.rot_dim = rot_dim;
  j.q_stride = query_row_stride;
  j.k_stride = key_row_stride;
  j.max_position = max_position;
  return pace::run_heads<false>(j, num_tokens, cache_dtype, is_neox != 0, dtype, stream,
                                "qk_norm_rotary_embedding");
}

extern "C" int pace_qk_norm_rotary_append(
    const int64_t* positions, void* query, const void* key, const void* value,
    const void* q_weight, const void* k_weight, float epsilon, int64_t num_tokens, int num_heads,
    int num_kv_heads, int head_size, int64_t query_row_stride, int64_t key_row_stride,
    int64_t value_row_stride, const void* cos_sin_cache, int cache_dtype, int rot_dim,
    int64_t max_position, int is_neox, void* paged_cache, int64_t num_pages, int page_size,
    const int64_t* slot_mapping, int32_t* bad_tokens, int dtype, cudaStream_t stream) {
  pace::HeadJob j = {};
  j.positions = positions;
  j.query = query;
  j.key = const_cast<void*>(key);
  j.value = value;
  j.q_weight = q_weight;
  j.k_weight = k_weight;
  j.cos_sin = cos_sin_cache;
  j.cache = paged_cache;
  j.slots = slot_mapping;
  j.bad = bad_tokens;
  j.eps = epsilon;
  j.num_tokens = (int)num_tokens;
  j.heads = num_heads;
  j.kv_heads = num_kv_heads;
  j.head_size = head_size;
  j.rot_dim = rot_dim;
  j.page_size = page_size;
  j.page_shift = page_size > 0 && (page_size & (page_size - 1)) == 0 ? __builtin_ctz(page_size) : -1;
  j.q_stride = query_row_stride;
  j.k_stride = key_row_stride;
  j.v_stride = value_row_stride;
  j.max_position = max_position;
  j.num_slots = num_pages < 0 || page_size <= 0 ? -1 : num_pages * page_size;
  return pace::run_heads<true>(j, num_tokens, cache_dtype, is_neox != 0, dtype, stream,
                               "qk_norm_rotary_append");
}
