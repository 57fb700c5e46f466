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
#include <algorithm>

#include "f32x2.cuh"
#include "tcgen05.cuh"

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
  float eps, share;  // share: 1 / head_size
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

// The same from shared memory.
template <typename C, int N>
__device__ __forceinline__ void shared_floats(const C* p, float* out) {
  if constexpr (sizeof(C) == 4) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const float4 v = *(reinterpret_cast<const float4*>(p) + i);
      out[4 * i] = v.x;
      out[4 * i + 1] = v.y;
      out[4 * i + 2] = v.z;
      out[4 * i + 3] = v.w;
    }
  } else {
    Traits<C>::unpack(*reinterpret_cast<const uint4*>(p), out);
  }
}

// The sum of a lane's squares.
template <int V>
__device__ __forceinline__ float squares(const float (&x)[V], const float (&y)[V]) {
  uint64_t sum = 0;
#pragma unroll
  for (int e = 0; e < V; e += 2) {
    const uint64_t a = two(x[e], x[e + 1]), b = two(y[e], y[e + 1]);
    sum = fma2(b, b, fma2(a, a, sum));
  }
  float lo, hi;
  apart(sum, lo, hi);
  return lo + hi;
}

// A lane's two vectors of a head, normalised and (turn) rotated.
template <int V, bool NEOX>
__device__ __forceinline__ void finish_head(float (&x)[V], float (&y)[V], const float (&wx)[V],
                                            const float (&wy)[V], const float (&c)[V],
                                            const float (&s)[V], float inv, bool turn) {
  const uint64_t f = two(inv, inv);
#pragma unroll
  for (int e = 0; e < V; e += 2) {
    apart(mul2(mul2(two(x[e], x[e + 1]), f), two(wx[e], wx[e + 1])), x[e], x[e + 1]);
    apart(mul2(mul2(two(y[e], y[e + 1]), f), two(wy[e], wy[e + 1])), y[e], y[e + 1]);
  }
  if (!turn) return;
  if constexpr (NEOX) {
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      const uint64_t a = two(x[e], x[e + 1]), b = two(y[e], y[e + 1]);
      const uint64_t co = two(c[e], c[e + 1]), si = two(s[e], s[e + 1]);
      apart(fma2(b, two(-s[e], -s[e + 1]), mul2(a, co)), x[e], x[e + 1]);
      apart(fma2(a, si, mul2(b, co)), y[e], y[e + 1]);
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

// G: lanes of a head.  NH: heads of a thread, of one token and one kind (query,
// key, value), which share the token's cosines and sines and the weight.
template <typename T, typename C, bool NEOX, bool APPEND, int G, int NH>
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(const HeadJob j) {
  using Tr = Traits<T>;
  constexpr int V = Tr::kVec;
  const int q_groups = (j.heads + NH - 1) / NH, kv_groups = (j.kv_heads + NH - 1) / NH;
  const int lanes = (q_groups + (APPEND ? 2 : 1) * kv_groups) * G;  // of a token
  const int64_t first = (int64_t)blockIdx.x * blockDim.x;
  const int64_t tok0 = first / lanes;
  const int at = (int)(first - tok0 * lanes) + (int)threadIdx.x;
  const int more = at / lanes;
  const int64_t tok = tok0 + more;
  const int group = (at - more * lanes) / G;
  const int l = threadIdx.x % G;
  const int units = j.head_size / (2 * V), turns = j.rot_dim / (2 * V);
  const bool live = tok < j.num_tokens && l < units;
  const bool is_q = group < q_groups, is_v = APPEND && group >= q_groups + kv_groups;
  const int h0 = (is_q ? group : is_v ? group - q_groups - kv_groups : group - q_groups) * NH;
  const int heads = is_q ? j.heads : j.kv_heads;
  // this lane's two vectors of a head
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
  row += (int64_t)h0 * j.head_size;
  pdl_launch_dependents();
  if (live) {
#pragma unroll
    for (int i = 0; i < NH; ++i)
      if (h0 + i < heads) {
        prefetch_line(row + i * j.head_size + d0);
        prefetch_line(row + i * j.head_size + d1);
      }
  }
  pdl_wait();
  uint4 xv[NH], yv[NH];
  int64_t pos = -1, slot = -1;
  if (live) {
#pragma unroll
    for (int i = 0; i < NH; ++i)
      if (h0 + i < heads) {
        xv[i] = ld_v4(row + i * j.head_size + d0);
        yv[i] = ld_v4(row + i * j.head_size + d1);
      }
    pos = j.positions[tok];
    if (APPEND && !is_q) slot = j.slots[tok];
  }
  const bool placed = pos >= 0 && pos < j.max_position;
  T* dst = row;
  bool store = live && placed;
  if (APPEND && !is_q && live) {
    store = goes_to_cache(j, slot, placed, l == 0 && group == q_groups);
    if (store)
      dst = static_cast<T*>(j.cache) +
            (cache_row(j, slot, is_v) * j.kv_heads + h0) * (int64_t)j.head_size;
  }
  float c[V], s[V], wx[V], wy[V];
  if (store && !is_v) {
    const T* weight = static_cast<const T*>(is_q ? j.q_weight : j.k_weight);
    load_floats<T, V>(weight + d0, wx);
    load_floats<T, V>(weight + d1, wy);
    if (turn) {
      const C* table = static_cast<const C*>(j.cos_sin) + pos * j.rot_dim + l * V;
      load_floats<C, V>(table, c);
      load_floats<C, V>(table + j.rot_dim / 2, s);
    }
  }
#pragma unroll
  for (int i = 0; i < NH; ++i) {
    const bool mine = h0 + i < heads;  // the same for a head's lanes
    float x[V], y[V], ss = 0.f;
    if (live && mine) {
      Tr::unpack(xv[i], x);
      Tr::unpack(yv[i], y);
      ss = squares<V>(x, y);
    }
#pragma unroll
    for (int m = 1; m < G; m <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
    if (!store || !mine) continue;
    if (!is_v) {
      const float inv = rsqrtf(ss * j.share + j.eps);
      finish_head<V, NEOX>(x, y, wx, wy, c, s, inv, turn);
      xv[i] = Tr::pack(x);
      yv[i] = Tr::pack(y);
    }
    st_v4(dst + i * j.head_size + d0, xv[i]);
    st_v4(dst + i * j.head_size + d1, yv[i]);
  }
}

// ------------------------------------------------------------ many tokens --
// A CTA walks tiles of a few neighbouring tokens with a ring of stages, each the
// tokens' query, key and value rows and their rows of the cos/sin table, brought in
// by bulk copies: warp 8 reads positions ahead and copies in, a token a lane; warps
// 0 to 7 normalise and rotate in place in shared memory; warp 9 copies the rows out
// (values untouched by any register).  So the bytes in flight are the ring's,
// whatever the registers, and the chain position, cosines, heads is off the
// critical path.  16384 tokens with the append: 64 + 8 heads of 128 111 us, 6.1 TB/s
// (the kernel for few tokens 141); 32 + 8 heads 71 us (87), in place 65 (74).
//
// A stage has tokens for up to 36 KB, since it costs about a microsecond beside its
// bytes (32 + 8 heads: one token 79 us, two 71).  A token is the work of two warps,
// four where it has a stage to itself: all eight warps on one token wait for one
// another's latency (64 + 8 heads: 130 us).
constexpr int kStreamWarps = 8, kStreamThreads = (kStreamWarps + 2) * 32;
constexpr int kStreamStages = 8;  // at most
constexpr int kStreamRing = 110 * 1024, kStreamTile = 36 * 1024;
constexpr uint64_t kWaitLimitNs = 1000000000ull;  // 1 s per wait
constexpr int32_t kFaultTimeout = 1 << 30;

struct StreamCtl {
  uint64_t full[kStreamStages], done[kStreamStages], empty[kStreamStages];
  uint32_t placed[kStreamStages];  // tokens of the stage that have a position, a bit each
  int abort;
};

struct StreamShape {
  int stages, tokens, share, token_bytes, q_bytes, kv_bytes, table_bytes;  // tokens: of a stage
};

__device__ __forceinline__ void bulk_in(void* dst, const void* src, int bytes, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          tc::smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(tc::smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void bulk_out(void* dst, const void* src, int bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst),
               "r"(tc::smem_u32(src)), "r"(bytes)
               : "memory");
}

template <typename T, typename C, bool NEOX, bool APPEND, int G>
__global__ void __launch_bounds__(kStreamThreads, 2)
    qk_norm_rope_stream_kernel(const HeadJob j, const StreamShape p, int32_t* fault) {
  using Tr = Traits<T>;
  constexpr int V = Tr::kVec;
  extern __shared__ __align__(128) uint8_t ring[];
  const int stage_bytes = p.tokens * p.token_bytes;
  StreamCtl* ctl = reinterpret_cast<StreamCtl*>(ring + p.stages * stage_bytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      tc::mbar_init(&ctl->full[s], 1);
      tc::mbar_init(&ctl->done[s], kStreamWarps);
      tc::mbar_init(&ctl->empty[s], 1);
    }
    ctl->abort = 0;
    tc::fence_barrier_init();
  }
  __syncthreads();
  pdl_launch_dependents();
  pdl_wait();
  auto wait = [&](uint64_t* bar, uint32_t parity) {  // by a whole warp
    const bool ok = tc::mbar_wait(bar, parity & 1u, kWaitLimitNs, &ctl->abort);
    if (__all_sync(0xffffffffu, ok)) return true;
    if (lane == 0) {
      *reinterpret_cast<volatile int*>(&ctl->abort) = 1;
      if (fault) atomicOr(fault, kFaultTimeout);
    }
    return false;
  };
  const int64_t step = (int64_t)gridDim.x * p.tokens;
  const int64_t first = (int64_t)blockIdx.x * p.tokens;
  if (warp == kStreamWarps) {
    // ---- copies in, a token a lane --------------------------------------------
    auto position = [&](int64_t tok0) -> int64_t {
      return lane < p.tokens && tok0 + lane < j.num_tokens ? j.positions[tok0 + lane] : -1;
    };
    int64_t pos = position(first);
    uint32_t i = 0;
    for (int64_t tok0 = first; tok0 < j.num_tokens; tok0 += step, ++i) {
      const uint32_t s = i % p.stages;
      const int64_t here = pos, tok = tok0 + lane;
      pos = position(tok0 + step);
      if (i >= (uint32_t)p.stages && !wait(&ctl->empty[s], i / p.stages - 1)) break;
      const bool placed = here >= 0 && here < j.max_position;
      const uint32_t mask = __ballot_sync(0xffffffffu, placed);
      if (lane == 0) {
        ctl->placed[s] = mask;
        tc::mbar_arrive_expect_tx(&ctl->full[s], (uint32_t)(__popc(mask) * p.token_bytes));
      }
      __syncwarp();
      if (placed) {
        uint8_t* st = ring + s * stage_bytes + lane * p.token_bytes;
        if (p.q_bytes)
          bulk_in(st, static_cast<const T*>(j.query) + tok * j.q_stride, p.q_bytes, &ctl->full[s]);
        if (p.kv_bytes)
          bulk_in(st + p.q_bytes, static_cast<const T*>(j.key) + tok * j.k_stride, p.kv_bytes,
                  &ctl->full[s]);
        if (APPEND)
          bulk_in(st + p.q_bytes + p.kv_bytes, static_cast<const T*>(j.value) + tok * j.v_stride,
                  p.kv_bytes, &ctl->full[s]);
        bulk_in(st + p.token_bytes - p.table_bytes,
                static_cast<const C*>(j.cos_sin) + here * j.rot_dim, p.table_bytes, &ctl->full[s]);
      }
    }
    // every copy has landed before the shared memory is given up
    for (uint32_t q = i > (uint32_t)p.stages ? i - p.stages : 0; q < i; ++q)
      tc::mbar_wait(&ctl->full[q % p.stages], (q / p.stages) & 1u, kWaitLimitNs, nullptr);
  } else if (warp == kStreamWarps + 1) {
    // ---- copies out, a token a lane -------------------------------------------
    auto slot_of = [&](int64_t tok0) -> int64_t {
      return APPEND && lane < p.tokens && tok0 + lane < j.num_tokens ? j.slots[tok0 + lane] : -1;
    };
    int64_t slot = slot_of(first);
    uint32_t i = 0;
    for (int64_t tok0 = first; tok0 < j.num_tokens; tok0 += step, ++i) {
      const uint32_t s = i % p.stages;
      const int64_t here = slot, tok = tok0 + lane;
      slot = slot_of(tok0 + step);
      if (!wait(&ctl->done[s], i / p.stages)) break;
      const uint8_t* st = ring + s * stage_bytes + lane * p.token_bytes;
      const bool placed = ctl->placed[s] >> lane & 1u;
      if (placed && p.q_bytes) bulk_out(static_cast<T*>(j.query) + tok * j.q_stride, st, p.q_bytes);
      if constexpr (APPEND) {
        if (goes_to_cache(j, here, placed, true)) {
          const int64_t row = (int64_t)j.kv_heads * j.head_size;
          T* cache = static_cast<T*>(j.cache);
          bulk_out(cache + cache_row(j, here, 0) * row, st + p.q_bytes, p.kv_bytes);
          bulk_out(cache + cache_row(j, here, 1) * row, st + p.q_bytes + p.kv_bytes, p.kv_bytes);
        }
      } else if (placed && p.kv_bytes) {
        bulk_out(static_cast<T*>(j.key) + tok * j.k_stride, st + p.q_bytes, p.kv_bytes);
      }
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      // the stage before this one has been read
      asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
      __syncwarp();
      if (lane == 0 && i > 0) tc::mbar_arrive(&ctl->empty[(i - 1) % p.stages]);
    }
    asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  } else {
    // ---- norm and rotation, in place --------------------------------------
    const int l = threadIdx.x % G;
    const int units = j.head_size / (2 * V), turns = j.rot_dim / (2 * V);
    const bool live = l < units, turn = l < turns;
    const int d0 = NEOX && turn ? l * V : l * 2 * V;
    const int d1 = NEOX && turn ? j.rot_dim / 2 + d0 : d0 + V;
    const int heads = j.heads + j.kv_heads;
    const int share = p.share;
    const uint32_t groups = kStreamWarps / share, group = warp / share;
    uint4 qx = make_uint4(0, 0, 0, 0), qy = qx, kx = qx, ky = qx;
    if (live) {
      const T *qw = static_cast<const T*>(j.q_weight), *kw = static_cast<const T*>(j.k_weight);
      qx = __ldg(reinterpret_cast<const uint4*>(qw + d0));
      qy = __ldg(reinterpret_cast<const uint4*>(qw + d1));
      kx = __ldg(reinterpret_cast<const uint4*>(kw + d0));
      ky = __ldg(reinterpret_cast<const uint4*>(kw + d1));
    }
    uint32_t i = 0;
    for (int64_t tok0 = first; tok0 < j.num_tokens; tok0 += step, ++i) {
      const uint32_t s = i % p.stages;
      if (!wait(&ctl->full[s], i / p.stages)) break;
      const uint32_t placed = ctl->placed[s];
      // p.share warps a token, each with the token's cosines in registers; a group of them takes
      // the next token whether or not it is in the same stage
      for (int t = 0; t < p.tokens; ++t) {
        if ((i * p.tokens + t) % groups != group || !(placed >> t & 1u)) continue;
        uint8_t* st = ring + s * stage_bytes + t * p.token_bytes;
        float c[V], sn[V];
        if (turn) {
          const C* table = reinterpret_cast<const C*>(st + p.token_bytes - p.table_bytes) + l * V;
          shared_floats<C, V>(table, c);
          shared_floats<C, V>(table + j.rot_dim / 2, sn);
        }
        // whole warps stay in the loop, for the shuffles
        for (int h0 = warp % share * (32 / G); h0 < heads; h0 += share * (32 / G)) {
          const int head = h0 + lane / G;
          const bool mine = live && head < heads;
          T* row = reinterpret_cast<T*>(st) + head * j.head_size;  // keys follow the queries
          float x[V], y[V], ss = 0.f;
          if (mine) {
            Tr::unpack(*reinterpret_cast<const uint4*>(row + d0), x);
            Tr::unpack(*reinterpret_cast<const uint4*>(row + d1), y);
            ss = squares<V>(x, y);
          }
#pragma unroll
          for (int m = 1; m < G; m <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
          if (!mine) continue;
          const float inv = rsqrtf(ss * j.share + j.eps);
          const bool is_q = head < j.heads;
          float wx[V], wy[V];
          Tr::unpack(is_q ? qx : kx, wx);
          Tr::unpack(is_q ? qy : ky, wy);
          finish_head<V, NEOX>(x, y, wx, wy, c, sn, inv, turn);
          *reinterpret_cast<uint4*>(row + d0) = Tr::pack(x);
          *reinterpret_cast<uint4*>(row + d1) = Tr::pack(y);
        }
      }
      // what the copies out read is written
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&ctl->done[s]);
    }
  }
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
    const float inv = rsqrtf(ss * j.share + j.eps);
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
int launch_heads(const HeadJob& j, int32_t* fault, cudaStream_t stream, const char* name) {
  constexpr int V = Traits<T>::kVec;
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
    const int64_t q_bytes = (int64_t)j.heads * j.head_size * sizeof(T);
    const int64_t kv_bytes = (int64_t)j.kv_heads * j.head_size * sizeof(T);
    const int64_t table_bytes = (int64_t)j.rot_dim * sizeof(C);
    const int64_t token_bytes = q_bytes + (APPEND ? 2 : 1) * kv_bytes + table_bytes;
    // Rows of 8 KB and more, and 64 MB of them (32 + 8 heads of 128 with the append: 2048 tokens
    // 14.1 us against 12.3, 4096 tokens 21.8 against 22.5; 24 heads of 64, 4 KB rows, 16384 tokens
    // 35 against 30)
    if (token_bytes >= 8192 && token_bytes <= kStreamRing / 3 &&
        token_bytes * j.num_tokens >= (64 << 20)) {
      int device = 0;
      if (cudaGetDevice(&device) != cudaSuccess) device = 0;
      const int tokens = 2 * token_bytes > kStreamTile ? 1 : 4 * token_bytes > kStreamTile ? 2 : 4;
      const StreamShape p{(int)std::min<int64_t>(kStreamStages, kStreamRing / (tokens * token_bytes)),
                          tokens,
                          tokens == 1 ? 4 : 2,
                          (int)token_bytes,
                          (int)q_bytes,
                          (int)kv_bytes,
                          (int)table_bytes};
      const int smem = p.stages * p.tokens * p.token_bytes + (int)sizeof(StreamCtl);
      const int ctas = (int)std::min<int64_t>(2 * sm_count(device), ceil_div(j.num_tokens, tokens));
      auto go = [&](auto kernel) {
        cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), device,
                                            kStreamRing + (int)sizeof(StreamCtl));
        if (e != cudaSuccess) return e;
        return launch(kernel, dim3((unsigned)ctas), dim3(kStreamThreads),
                      (size_t)smem, stream, j, p, fault);
      };
      switch (g) {
        case 1: err = go(qk_norm_rope_stream_kernel<T, C, NEOX, APPEND, 1>); break;
        case 2: err = go(qk_norm_rope_stream_kernel<T, C, NEOX, APPEND, 2>); break;
        case 4: err = go(qk_norm_rope_stream_kernel<T, C, NEOX, APPEND, 4>); break;
        case 8: err = go(qk_norm_rope_stream_kernel<T, C, NEOX, APPEND, 8>); break;
        case 16: err = go(qk_norm_rope_stream_kernel<T, C, NEOX, APPEND, 16>); break;
        default: err = go(qk_norm_rope_stream_kernel<T, C, NEOX, APPEND, 32>); break;
      }
      return err == cudaSuccess ? PACE_OK : cuda_fail(err, name);
    }
    // Two heads a thread above 256 tokens (512 tokens of 32 + 8 heads in place: 4.2 us with one, 3.2
    // with two, 4.3 with four; 64 tokens with the append 2.0, 2.2 and 2.8)
    const int nh = j.num_tokens > 256 ? 2 : 1;
    constexpr int kThreads = 128;
    const int groups =
        (int)(ceil_div(j.heads, nh) + (APPEND ? 2 : 1) * ceil_div(j.kv_heads, nh));
    const int64_t ctas = ceil_div((int64_t)j.num_tokens * groups * g, kThreads);
    if (ctas > INT32_MAX) return fail(PACE_ERR_TOO_LARGE, "%s: too many heads", name);
    auto go = [&](auto one, auto two) {
      return launch(nh == 1 ? one : two, dim3((unsigned)ctas), dim3(kThreads), 0, stream, j);
    };
#define PACE_HEADS_CASE(LANES)                           \
  go(qk_norm_rope_kernel<T, C, NEOX, APPEND, LANES, 1>, \
     qk_norm_rope_kernel<T, C, NEOX, APPEND, LANES, 2>)
    switch (g) {
      case 1: err = PACE_HEADS_CASE(1); break;
      case 2: err = PACE_HEADS_CASE(2); break;
      case 4: err = PACE_HEADS_CASE(4); break;
      case 8: err = PACE_HEADS_CASE(8); break;
      case 16: err = PACE_HEADS_CASE(16); break;
      default: err = PACE_HEADS_CASE(32); break;
    }
#undef PACE_HEADS_CASE
  } else {
    err = launch(qk_norm_rope_scalar_kernel<T, C, NEOX, APPEND>, dim3((unsigned)j.num_tokens),
                 dim3(128), 0, stream, j);
  }
  return err == cudaSuccess ? PACE_OK : cuda_fail(err, name);
}

template <bool APPEND>
int run_heads(const HeadJob& j, int64_t num_tokens, int cache_dtype, bool neox, int dtype,
              int32_t* fault, cudaStream_t stream, const char* name) {
  if (num_tokens < 0 || num_tokens > INT32_MAX || j.heads < 0 || j.kv_heads < 0 ||
      j.head_size <= 0 || (j.heads + 2 * (int64_t)j.kv_heads) * j.head_size > (1 << 30))
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
      return neox ? launch_heads<scalar_t, float, true, APPEND>(j, fault, stream, name)
                  : launch_heads<scalar_t, float, false, APPEND>(j, fault, stream, name);
    if (cache_dtype == dtype)
      return neox ? launch_heads<scalar_t, scalar_t, true, APPEND>(j, fault, stream, name)
                  : launch_heads<scalar_t, scalar_t, false, APPEND>(j, fault, stream, name);
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
    int rot_dim, int64_t max_position, int is_neox, int dtype, int32_t* fault_flags,
    cudaStream_t stream) {
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
  j.share = 1.f / (float)head_size;
  j.rot_dim = rot_dim;
  j.q_stride = query_row_stride;
  j.k_stride = key_row_stride;
  j.max_position = max_position;
  return pace::run_heads<false>(j, num_tokens, cache_dtype, is_neox != 0, dtype, fault_flags, stream,
                                "qk_norm_rotary_embedding");
}

extern "C" int pace_qk_norm_rotary_append(
    const int64_t* positions, void* query, const void* key, const void* value,
    const void* q_weight, const void* k_weight, float epsilon, int64_t num_tokens, int num_heads,
    int num_kv_heads, int head_size, int64_t query_row_stride, int64_t key_row_stride,
    int64_t value_row_stride, const void* cos_sin_cache, int cache_dtype, int rot_dim,
    int64_t max_position, int is_neox, void* paged_cache, int64_t num_pages, int page_size,
    const int64_t* slot_mapping, int32_t* bad_tokens, int dtype, int32_t* fault_flags,
    cudaStream_t stream) {
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
  j.share = 1.f / (float)head_size;
  j.rot_dim = rot_dim;
  j.page_size = page_size;
  j.page_shift = page_size > 0 && (page_size & (page_size - 1)) == 0 ? __builtin_ctz(page_size) : -1;
  j.q_stride = query_row_stride;
  j.k_stride = key_row_stride;
  j.v_stride = value_row_stride;
  j.max_position = max_position;
  j.num_slots = num_pages < 0 || page_size <= 0 ? -1 : num_pages * page_size;
  return pace::run_heads<true>(j, num_tokens, cache_dtype, is_neox != 0, dtype, fault_flags, stream,
                               "qk_norm_rotary_append");
}
