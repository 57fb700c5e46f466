// Products of 8-bit integers with a scale for each token and each output
// channel, for sm_100a: the projections of a decoder layer with 8-bit weights.
//
//   y_tn = (sum_k c_tk w_nk) * s_t * s_n  (+ bias_n) (+ residual_tn)
//   gate_up_silu:  silu(y_tn) * y_t(I + n),   weight [2 I, K]
//
// The sum is int32, so it is exact and the same in every order of its terms (K is
// at most 131071, where 128 * 128 * K still fits); the rest is fp32, rounded once.
//
// Three kernels on the tensor cores, all TMA (128-byte K blocks, 128-byte swizzle)
// into a ring, one thread issuing tcgen05.mma.kind::i8, and eight warps that drain
// the accumulator in TMEM through the scales:
//  * int8_gemm_kernel, many tokens, bound by the matrix rate: tokens in the
//    accumulator's rows, 256 on a CTA pair (cta_group::2), by up to 256 channels;
//  * int8_mid_kernel, 33 to 128 tokens, or more where whole tiles of the former
//    would leave half of the SMs idle: K cut over the CTAs of a cluster;
//  * int8_slice_kernel, up to 32 tokens, where the weight's bytes bound it: 32
//    channels a tile, so that there are tiles for all SMs without cutting one over
//    CTAs.  The 128 rows of the matrix instruction hold the channels' K in four
//    slices, its columns the tokens' K in the same slices: the four blocks where
//    the slices agree are partial sums, the others are not read.
//
// What TMA cannot take (a row stride or an address that is no multiple of 16 bytes)
// runs through registers and small matrix instructions (int8_dot_kernel).
#include <algorithm>
#include <type_traits>

#include "tcgen05.cuh"

namespace pace {
namespace {

constexpr int BK = 128;  // bytes of K per stage: one swizzle atom
constexpr int BM = 128;
constexpr int EPI_WARPS = 8;
constexpr int THREADS = (EPI_WARPS + 2) * 32;
constexpr int MAX_STAGES = 10;
constexpr int kRingBytes = 196608;  // at most
constexpr int kSmem = kRingBytes + 1024 + 256;
constexpr int kEpiBarrier = 1;
constexpr int CH = 16;  // columns drained at a time
constexpr uint64_t kWaitLimitNs = 1000000000ull;  // 1 s per wait
constexpr int32_t kFaultTimeout = 1 << 30;
constexpr int64_t kMaxK = 131071;
constexpr int64_t kMaxRows = 1 << 29;  // tokens, and channels: twice as many fit an int

struct Ctl {
  uint64_t full[MAX_STAGES];
  uint64_t empty[MAX_STAGES];
  uint64_t tmem_full[2];
  uint64_t tmem_empty[2];
  uint64_t drain;
  uint32_t tmem;
  int abort;
};
static_assert(sizeof(Ctl) <= 256, "");

struct GemmJob {
  void* out;
  const void* add;   // residual, or null
  const void* bias;  // or null
  const float *token_scales, *channel_scales;
  int64_t out_stride, add_stride;
  int tokens, channels;  // channels: output columns (half the weight's rows with SiLU)
  int k_blocks;
  int deep;        // whole K blocks: the tensor maps have them as a third axis
  int vec;         // out (and add) take 16-byte accesses
  int scales_vec;  // the channels' scales do
};

// Instruction descriptor of tcgen05.mma.kind::i8: int32 accumulator (bits 4-5 =
// 2), A and B signed (bits 7-9 and 10-12 = 1), both K-major, N >> 3, M >> 4.
__host__ __device__ constexpr uint32_t idesc_i8(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(m >> 4) << 24);
}

template <bool PAIR>
__device__ __forceinline__ void umma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                        uint32_t accumulate) {
  if constexpr (PAIR)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}

// 8 consecutive columns of this thread's TMEM lane; valid after tc::tmem_wait_ld.
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7])
      : "r"(taddr)
      : "memory");
}

// The box of rows y .. of the K blocks z .. of a three-axis map (bytes of a block,
// rows, blocks), in shared memory block by block; see make_map.
__device__ __forceinline__ void tma_load_deep(void* dst, const CUtensorMap* map, int32_t y,
                                              int32_t z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(tc::smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(y), "r"(z), "r"(tc::smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void tma_load_deep_pair(void* dst, const CUtensorMap* map, int32_t y,
                                                   int32_t z, uint32_t bar_cluster) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(tc::smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(y), "r"(z), "r"(bar_cluster)
      : "memory");
}

// Pulls a box of a tensor map into L2.
__device__ __forceinline__ void prefetch_deep(const CUtensorMap* map, int32_t y, int32_t z) {
  asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global.tile [%0, {%1, %2, %3}];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(0), "r"(y), "r"(z)
               : "memory");
}
__device__ __forceinline__ void prefetch_box(const CUtensorMap* map, int32_t x, int32_t y) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y)
               : "memory");
}

// Tile t's place: groups of kGroup rows of tiles, and within a group the rows
// fastest, so that the tiles in work at one time are about as many tokens high as
// channels wide and read little besides one another's operands.
constexpr int kGroup = 8;
__device__ __forceinline__ void place_of(int64_t t, int m_tiles, int n_tiles, int& mt, int& nt) {
  const int64_t group = (int64_t)kGroup * n_tiles;
  const int first = (int)(t / group) * kGroup;
  const int rows = min(kGroup, m_tiles - first);
  const int r = (int)(t - (int64_t)first * n_tiles);
  nt = r / rows;
  mt = first + r - nt * rows;
}

__device__ __forceinline__ void raise_fault(Ctl* ctl, int32_t* fault) {
  *reinterpret_cast<volatile int*>(&ctl->abort) = 1;
  if (fault) atomicOr(fault, kFaultTimeout);
}

__device__ __forceinline__ void epi_sync() {
  asm volatile("bar.sync %0, %1;" ::"n"(kEpiBarrier), "n"(EPI_WARPS * 32) : "memory");
}
__device__ __forceinline__ bool epi_all(bool pred) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "bar.red.and.pred q, %2, %3, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(pred ? 1u : 0u), "n"(kEpiBarrier), "n"(EPI_WARPS * 32)
      : "memory");
  return r != 0;
}

// 16-bit outputs take the approximate exponential and quotient, float32 the
// library's.  The approximate exponential's argument is rounded, which leaves an error
// that goes with |g|: at most (4 |g| + 16) 2^-24 of the value.  Where 1 + e^-g passes
// 2^126 (e^-g 2^128 in float32) the quotient is 0; what is lost is below |g| |u| 2^-126.
template <typename T>
__device__ __forceinline__ float silu_mul(float g, float u) {
  if constexpr (sizeof(T) == 2) return __fdividef(g, 1.f + __expf(-g)) * u;
  return g / (1.f + expf(-g)) * u;
}

// Scales of CH consecutive channels (those past the last are never used).
__device__ __forceinline__ void load_scales(const GemmJob& j, int n, float (&s)[CH]) {
  const int rows = n < j.channels ? j.channels : 2 * j.channels;
  if (j.scales_vec && n + CH <= rows) {
#pragma unroll
    for (int i = 0; i < CH / 4; ++i) {
      const float4 v = __ldg(reinterpret_cast<const float4*>(j.channel_scales + n) + i);
      s[4 * i] = v.x;
      s[4 * i + 1] = v.y;
      s[4 * i + 2] = v.z;
      s[4 * i + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int e = 0; e < CH; ++e) s[e] = __ldg(j.channel_scales + min(n + e, rows - 1));
  }
}

// CH consecutive channels n .. of one token in 16-byte accesses: add, round, store.
template <typename T>
__device__ __forceinline__ void put_channels(const GemmJob& j, int64_t t, int n, float* y) {
  constexpr int V = Traits<T>::kVec;
  T* o = static_cast<T*>(j.out) + t * j.out_stride + n;
  const T* add = j.add ? static_cast<const T*>(j.add) + t * j.add_stride + n : nullptr;
  if (n + CH <= j.channels) {
    if (add) {
#pragma unroll
      for (int i = 0; i < CH / V; ++i) {
        float f[V];
        Traits<T>::unpack(ld_v4(add + i * V), f);
#pragma unroll
        for (int e = 0; e < V; ++e) y[i * V + e] += f[e];
      }
    }
    if constexpr (CH % (2 * V) == 0) {
      if ((reinterpret_cast<uintptr_t>(o) & 31u) == 0) {  // whole sectors
#pragma unroll
        for (int i = 0; i < CH / (2 * V); ++i)
          st_v8(o + i * 2 * V, Traits<T>::pack(y + i * 2 * V), Traits<T>::pack(y + i * 2 * V + V));
        return;
      }
    }
#pragma unroll
    for (int i = 0; i < CH / V; ++i) st_v4(o + i * V, Traits<T>::pack(y + i * V));
  } else {
#pragma unroll
    for (int e = 0; e < CH; ++e)
      if (n + e < j.channels)
        o[e] = Traits<T>::from_f(add ? y[e] + Traits<T>::to_f(add[e]) : y[e]);
  }
}

// The same of a warp's 32 tokens t0 .., a token a lane, in single elements: by way of shared memory,
// so that 16 lanes take neighbouring channels of a token (512 tokens, K 4096, 4095 channels 17.1 us,
// a lane its own token 31.2; 2048 tokens, 32001 channels 228 and 716).
constexpr int kTurnPitch = CH + 1, kTurn = EPI_WARPS * 32 * kTurnPitch * (int)sizeof(float);
template <typename T>
__device__ __forceinline__ void put_turned(const GemmJob& j, int t0, int n, const float (&y)[CH],
                                           float* turn) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int e = 0; e < CH; ++e) turn[lane * kTurnPitch + e] = y[e];
  __syncwarp();
  constexpr int kRows = 32 / CH;  // at a time
  const int e = lane % CH, r0 = lane / CH;
  const int rows = n + e < j.channels ? min(32, j.tokens - t0) : 0;
  float v[32 / kRows];
#pragma unroll
  for (int i = 0; i < 32 / kRows; ++i) {
    const int r = r0 + i * kRows;
    v[i] = turn[r * kTurnPitch + e];
    if (j.add && r < rows)
      v[i] += Traits<T>::to_f(static_cast<const T*>(j.add)[(int64_t)(t0 + r) * j.add_stride + n + e]);
  }
#pragma unroll
  for (int i = 0; i < 32 / kRows; ++i) {
    const int r = r0 + i * kRows;
    if (r < rows)
      static_cast<T*>(j.out)[(int64_t)(t0 + r) * j.out_stride + n + e] = Traits<T>::from_f(v[i]);
  }
  __syncwarp();
}

// Four consecutive channels n .. of one token, as put_channels.
template <typename T>
__device__ __forceinline__ void put_four(const GemmJob& j, int64_t t, int n, bool all, float* y) {
  T* o = static_cast<T*>(j.out) + t * j.out_stride + n;
  const T* add = j.add ? static_cast<const T*>(j.add) + t * j.add_stride + n : nullptr;
  if (j.vec && all) {
    using Four = std::conditional_t<sizeof(T) == 2, uint2, uint4>;
    union {
      Four v;
      T x[4];
    } f;
    if (add) {
      f.v = *reinterpret_cast<const Four*>(add);
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] += Traits<T>::to_f(f.x[e]);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) f.x[e] = Traits<T>::from_f(y[e]);
    *reinterpret_cast<Four*>(o) = f.v;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < j.channels)
        o[e] = Traits<T>::from_f(add ? y[e] + Traits<T>::to_f(add[e]) : y[e]);
  }
}

// Tiles of the rows kernel: bn channels (gate and up together with SiLU), `sub` K
// blocks a ring stage.  From tile `whole` on they are done in two halves.
struct Tiling {
  int bn, sub, stages, m_tiles, n_tiles;
  int64_t whole;
};

// A pair's piece of work: a tile, or the half of one that starts `part` half widths in.
struct Piece {
  int mt, nt, half, part;
};
__device__ __forceinline__ Piece piece_of(int64_t i, const Tiling& p) {
  Piece w;
  const int64_t past = i - p.whole;
  w.half = past >= 0;
  w.part = w.half ? (int)past & 1 : 0;
  place_of(w.half ? p.whole + (past >> 1) : i, p.m_tiles, p.n_tiles, w.mt, w.nt);
  return w;
}

// One lane of the warp, the same in every call of the same warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r != 0;
}

// tc::mbar_wait with the clock read only when a wait is long.
__device__ __forceinline__ bool ring_wait(uint64_t* bar, uint32_t parity, Ctl* ctl) {
#pragma unroll 1
  for (int i = 0; i < 64; ++i)
    if (tc::mbar_try_wait(bar, parity)) return true;
  return tc::mbar_wait(bar, parity, kWaitLimitNs, &ctl->abort);
}

// A ring position: the stage, and the parity of the phase that its barriers wait for.
struct Turn {
  int s = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int stages) {
    if (++s == stages) {
      s = 0;
      phase ^= 1u;
    }
  }
};

// 256 tokens a CTA pair: the leader's 128 in its accumulator, its partner's in its
// own; each stages its tokens and half of the tile's channels.
template <typename T, bool SILU>
__global__ void __launch_bounds__(THREADS, 1)
    int8_gemm_kernel(const __grid_constant__ CUtensorMap tm_a,
                     const __grid_constant__ CUtensorMap tm_b,
                     const __grid_constant__ CUtensorMap tm_half, const GemmJob j, const Tiling p,
                     int32_t* fault) {
  constexpr int kA = BM * BK, kTmem = 512;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* tiles = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  Ctl* ctl = reinterpret_cast<Ctl*>(tiles + kRingBytes);
  const int nst = p.stages, bn = p.bn, sub = p.sub, out_cols = SILU ? bn / 2 : bn;
  const int kB = bn / 2 * BK, sb = kA + kB;  // bytes of a whole tile's K block in this CTA
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = tc::cluster_rank();
  const int workers = (int)gridDim.x >> 1;
  const int64_t t_first = blockIdx.x >> 1;
  const int64_t t_end = 2 * ((int64_t)p.m_tiles * p.n_tiles) - p.whole;

  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int s = 0; s < nst; ++s) {
      tc::mbar_init(&ctl->full[s], 1);
      tc::mbar_init(&ctl->empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      tc::mbar_init(&ctl->tmem_full[b], 1);
      tc::mbar_init(&ctl->tmem_empty[b], 2 * EPI_WARPS);
    }
    tc::mbar_init(&ctl->drain, 1);
    ctl->abort = 0;
    tc::fence_barrier_init();
  }
  if (warp == EPI_WARPS && lane == 0) {
    tc::tma_prefetch_desc(&tm_a);
    tc::tma_prefetch_desc(&tm_b);
    tc::tma_prefetch_desc(&tm_half);
  }
  if (warp == 0) tc::tmem_alloc_pair(&ctl->tmem, kTmem);
  tc::tc_fence_before();
  __syncthreads();
  tc::cluster_sync();
  tc::tc_fence_after();
  const uint32_t tmem = ctl->tmem;
  pdl_wait();

  if (warp == EPI_WARPS) {
    // ---- TMA producer: the whole warp walks, one lane issues ------------------
    const bool issues = elect_one();
    int64_t i = 0;
    bool ok = true;
    Turn turn;
    // both CTAs' copies complete on the leader's barrier, which expects the bytes of both
    const uint32_t full0 = tc::map_to_rank(&ctl->full[0], 0);
    for (int64_t t = t_first; ok && t < t_end; t += workers) {
      const Piece w = piece_of(t, p);
      const CUtensorMap* tm_w = w.half ? &tm_half : &tm_b;
      const int a0 = (2 * w.mt + (int)rank) * BM, kW = kB >> w.half;
      // with SiLU the leader has the gate's rows, its partner the up's
      const int b0 = w.nt * out_cols + w.part * (out_cols / 2) +
                     (int)rank * (SILU ? j.channels : bn / 2 >> w.half);
      for (int kb = 0; kb < j.k_blocks; kb += sub, ++i) {
        const int s = turn.s;
        if (i >= nst && !ring_wait(&ctl->empty[s], turn.phase ^ 1u, ctl)) {
          ok = false;
          break;
        }
        if (issues) {
          uint8_t* a = tiles + s * sub * sb;
          uint8_t* b = a + sub * kA;
          const uint32_t bar = full0 + (uint32_t)(s * sizeof(uint64_t));
          if (rank == 0) tc::mbar_arrive_expect_tx(&ctl->full[s], 2 * sub * (kA + kW));
          if (j.deep) {
            tma_load_deep_pair(a, &tm_a, a0, kb, bar);
            tma_load_deep_pair(b, tm_w, b0, kb, bar);
          } else {
            for (int u = 0; u < sub; ++u) {
              tc::tma_load_2d_pair(a + u * kA, &tm_a, (kb + u) * BK, a0, bar);
              tc::tma_load_2d_pair(b + u * kW, tm_w, (kb + u) * BK, b0, bar);
            }
          }
        }
        __syncwarp();
        turn.next(nst);
      }
    }
    if (!ok && lane == 0) raise_fault(ctl, fault);
    // every copy has landed before the shared memory is given up; the partner leaves after the
    // leader, at the closing cluster barrier
    if (rank == 0)
      for (int64_t q = i > nst ? i - nst : 0; q < i; ++q)
        tc::mbar_wait(&ctl->full[q % nst], (uint32_t)(q / nst) & 1u, kWaitLimitNs, nullptr);
  } else if (warp == EPI_WARPS + 1) {
    // ---- MMA issuer, in the leader ------------------------------------------
    if (rank == 0) {
      const bool issues = elect_one();
      int n = 0;
      bool ok = true;
      Turn turn;
      for (int64_t t = t_first; ok && t < t_end; t += workers, ++n) {
        const int half = t >= p.whole, kW = kB >> half;
        const uint32_t idesc = idesc_i8(2 * BM, bn >> half);
        const int b = n & 1;
        const uint32_t use_b = (uint32_t)(n >> 1);
        if (use_b > 0 &&
            !tc::mbar_wait(&ctl->tmem_empty[b], (use_b - 1) & 1u, kWaitLimitNs, &ctl->abort)) {
          ok = false;
          break;
        }
        tc::tc_fence_after();
        const uint32_t d = tmem + (uint32_t)(b * 256);
        for (int kb = 0; kb < j.k_blocks; kb += sub) {
          const int s = turn.s;
          if (!ring_wait(&ctl->full[s], turn.phase, ctl)) {
            ok = false;
            break;
          }
          tc::tc_fence_after();
          if (issues) {
            const uint32_t a_addr = tc::smem_u32(tiles + s * sub * sb);
            uint64_t ad = tc::umma_desc_sw128(a_addr);
            uint64_t bd = tc::umma_desc_sw128(a_addr + sub * kA);
            for (int u = 0; u < sub; ++u) {  // blocks past K are zero
#pragma unroll
              for (int k = 0; k < BK / 32; ++k)
                umma_i8<true>(d, ad + 2 * k, bd + 2 * k, idesc, kb > 0 || u > 0 || k > 0 ? 1u : 0u);
              ad += kA >> 4;
              bd += (uint64_t)kW >> 4;
            }
            tc::umma_commit_pair_both(&ctl->empty[s]);
          }
          __syncwarp();
          turn.next(nst);
        }
        if (ok && issues) tc::umma_commit_pair_both(&ctl->tmem_full[b]);
        __syncwarp();
      }
      if (!ok && lane == 0) raise_fault(ctl, fault);
      // every MMA has completed before TMEM is freed
      if (issues) tc::umma_commit_pair(&ctl->drain);
      tc::mbar_wait(&ctl->drain, 0, kWaitLimitNs, nullptr);
    }
  } else {
    // ---- epilogue: warp w drains lanes 32 (w % 4) .. +31, half w / 4 of the columns --------
    const int row = (warp % 4) * 32 + lane;
    const uint32_t tmem_empty0 = tc::map_to_rank(&ctl->tmem_empty[0], 0);
    float* turn = reinterpret_cast<float*>(ctl + 1) + warp * 32 * kTurnPitch;  // unless j.vec
    int n = 0;
    for (int64_t t = t_first; t < t_end; t += workers, ++n) {
      const int b = n & 1;
      const Piece w = piece_of(t, p);
      const int m = (2 * w.mt + (int)rank) * BM + row;  // this thread's token
      const int c0 = w.nt * out_cols + w.part * (out_cols / 2);  // the piece's first channel
      const int cols = out_cols / 2 >> w.half;                   // of this warp
      const int c_begin = (warp / 4) * cols, c_end = c_begin + cols;
      const int up = bn / 2 >> w.half;  // SiLU: the up columns' distance
      const bool valid = m < j.tokens;
      const float s_row = valid ? j.token_scales[m] : 0.f;
      bool ready = tc::mbar_wait(&ctl->tmem_full[b], (uint32_t)(n >> 1) & 1u, kWaitLimitNs,
                                 &ctl->abort);
      ready = epi_all(ready);
      if (!ready) {
        raise_fault(ctl, fault);
        break;
      }
      tc::tc_fence_after();
      const uint32_t acc = tmem + (uint32_t)(b * 256) + ((uint32_t)(warp % 4 * 32) << 16);
#pragma unroll 1
      for (int c = c_begin; c < c_end && c0 + c < j.channels; c += CH) {
        __syncwarp();
        uint32_t r[CH], r2[CH];
        tc::tmem_ld16(acc + (uint32_t)c, r);
        if (SILU) tc::tmem_ld16(acc + (uint32_t)(c + up), r2);
        const int ch = c0 + c;
        float sc[CH], sc2[CH];
        load_scales(j, ch, sc);
        if (SILU) load_scales(j, j.channels + ch, sc2);
        tc::tmem_wait_ld(r);
        if (SILU) tc::tmem_wait_ld(r2);
        if (valid || !j.vec) {
          float y[CH];
#pragma unroll
          for (int e = 0; e < CH; ++e) {
            y[e] = (float)(int)r[e] * s_row * sc[e];
            if (SILU) y[e] = silu_mul<T>(y[e], (float)(int)r2[e] * s_row * sc2[e]);
          }
          if (!SILU && j.bias) {
            const T* bias = static_cast<const T*>(j.bias);
#pragma unroll
            for (int e = 0; e < CH; ++e) y[e] += Traits<T>::to_f(bias[min(ch + e, j.channels - 1)]);
          }
          if (j.vec)
            put_channels<T>(j, m, ch, y);
          else
            put_turned<T>(j, m - lane, ch, y, turn);
        }
      }
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive_cluster(tmem_empty0 + (uint32_t)(b * sizeof(uint64_t)));
    }
  }

  tc::tc_fence_before();
  __syncthreads();
  // neither CTA leaves (nor frees TMEM) while its partner may still signal its barriers or read its
  // shared memory
  tc::cluster_sync();
  if (warp == 0) tc::tmem_dealloc_pair(tmem, kTmem);
}

// ------------------------------------------------------------- few tokens --
// 32 channels a tile.  Quarter q of the accumulator's rows holds them over slice
// q of K; with SiLU quarters 0 and 1 the gate's two slices, 2 and 3 the up's.  The
// columns hold the tokens, `tc` (a multiple of 8) for each slice.  So row quarter q
// and column group (q mod slices) belong to one slice; the other blocks of the
// accumulator are products of different slices and stay unread.  That costs matrix
// rate, of which there is enough (32 tokens: an instruction a K block is 128 columns
// wide, 64 bytes of weight a clock and SM, where memory delivers 23), and saves a
// reduction over CTAs: the slices are summed through shared memory.  The ring is small enough for two CTAs an SM, so that the
// next kernel's CTAs start, and pull their first weights into L2, beside this one's.
// Each takes at most half of TMEM; the kernels that take all of it have over 160 KB of
// shared memory, so none of their CTAs can wait beside one of these for its columns.
constexpr int kSliceCh = 32, kSliceTok = 16;  // of a tile; of a pass through shared memory
constexpr int kSliceRing = 98304;
constexpr int kSliceAhead = 12;  // blocks that are pulled into L2 before the wait
constexpr int kSliceSum = 4 * kSliceCh * kSliceTok * 4;
constexpr int kSliceRest = kSliceSum + 1024 + 256;

struct SliceTiling {
  int tc, stages, ring, tmem_cols, tiles, slice_blocks;
};

template <typename T, bool SILU>
__global__ void __launch_bounds__(THREADS, 2)
    int8_slice_kernel(const __grid_constant__ CUtensorMap tm_w,
                      const __grid_constant__ CUtensorMap tm_x, const GemmJob j,
                      const SliceTiling p, int32_t* fault) {
  constexpr int SL = SILU ? 2 : 4, kA = BM * BK, kBox = kSliceCh * BK;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* tiles = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  int32_t* sums = reinterpret_cast<int32_t*>(tiles + p.ring);  // [quarter][token][channel]
  Ctl* ctl = reinterpret_cast<Ctl*>(tiles + p.ring + kSliceSum);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sb = kA + SL * p.tc * BK, cols = SL * p.tc;

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      tc::mbar_init(&ctl->full[s], 1);
      tc::mbar_init(&ctl->empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      tc::mbar_init(&ctl->tmem_full[b], 1);
      tc::mbar_init(&ctl->tmem_empty[b], EPI_WARPS);
    }
    tc::mbar_init(&ctl->drain, 1);
    ctl->abort = 0;
    tc::fence_barrier_init();
  }
  // The weight's boxes of quarter q: channels of tile t (the up's with SiLU from quarter 2 on)
  auto w_row = [&](int t, int q) { return t * kSliceCh + (SILU && q >= SL ? j.channels : 0); };
  auto w_col = [&](int kb, int q) { return (kb * SL + q % SL) * BK; };
  if (warp == EPI_WARPS && lane == 0) {
    tc::tma_prefetch_desc(&tm_w);
    tc::tma_prefetch_desc(&tm_x);
    // L2 is the point of coherence: what an earlier kernel still writes to the weight is read from
    // there after the wait
    for (int kb = 0; kb < min(p.slice_blocks, kSliceAhead); ++kb)
      for (int q = 0; q < 4; q += j.deep ? SL : 1) {
        if (j.deep)
          prefetch_deep(&tm_w, w_row((int)blockIdx.x, q), kb * SL);
        else
          prefetch_box(&tm_w, w_col(kb, q), w_row((int)blockIdx.x, q));
      }
  }
  if (warp == 0) tc::tmem_alloc(&ctl->tmem, (uint32_t)p.tmem_cols);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = ctl->tmem;
  pdl_launch_dependents();
  pdl_wait();

  if (warp == EPI_WARPS) {
    // ---- TMA producer: the whole warp walks, one lane issues ------------------
    {
      const bool issues = elect_one();
      int64_t i = 0;
      bool ok = true;
      Turn turn;
      for (int t = blockIdx.x; ok && t < p.tiles; t += gridDim.x) {
        for (int kb = 0; kb < p.slice_blocks; ++kb, ++i) {
          const int s = turn.s;
          if (i >= p.stages && !ring_wait(&ctl->empty[s], turn.phase ^ 1u, ctl)) {
            ok = false;
            break;
          }
          if (issues) {
            uint8_t* a = tiles + s * sb;
            tc::mbar_arrive_expect_tx(&ctl->full[s], (uint32_t)sb);
            if (j.deep) {
#pragma unroll
              for (int q = 0; q < 4; q += SL)
                tma_load_deep(a + q * kBox, &tm_w, w_row(t, q), kb * SL, &ctl->full[s]);
              tma_load_deep(a + kA, &tm_x, 0, kb * SL, &ctl->full[s]);
            } else {
#pragma unroll
              for (int q = 0; q < 4; ++q)
                tc::tma_load_2d(a + q * kBox, &tm_w, w_col(kb, q), w_row(t, q), &ctl->full[s]);
#pragma unroll
              for (int q = 0; q < SL; ++q)
                tc::tma_load_2d(a + kA + q * p.tc * BK, &tm_x, w_col(kb, q), 0, &ctl->full[s]);
            }
          }
          __syncwarp();
          turn.next(p.stages);
        }
      }
      if (!ok && lane == 0) raise_fault(ctl, fault);
      for (int64_t q = i > p.stages ? i - p.stages : 0; q < i; ++q)
        tc::mbar_wait(&ctl->full[q % p.stages], (uint32_t)(q / p.stages) & 1u, kWaitLimitNs, nullptr);
    }
  } else if (warp == EPI_WARPS + 1) {
    // ---- MMA issuer ---------------------------------------------------------
    {
      const bool issues = elect_one();
      const uint32_t idesc = idesc_i8(BM, cols);
      int n = 0;
      bool ok = true;
      Turn turn;
      for (int t = blockIdx.x; ok && t < p.tiles; t += gridDim.x, ++n) {
        const int b = n & 1, use = n >> 1;
        if (use > 0 && !tc::mbar_wait(&ctl->tmem_empty[b], (uint32_t)(use - 1) & 1u, kWaitLimitNs,
                                      &ctl->abort)) {
          ok = false;
          break;
        }
        tc::tc_fence_after();
        const uint32_t d = tmem + (uint32_t)(b * cols);
        for (int kb = 0; kb < p.slice_blocks; ++kb) {
          const int s = turn.s;
          if (!ring_wait(&ctl->full[s], turn.phase, ctl)) {
            ok = false;
            break;
          }
          tc::tc_fence_after();
          if (issues) {
            const uint32_t a_addr = tc::smem_u32(tiles + s * sb);
            const uint64_t ad = tc::umma_desc_sw128(a_addr);
            const uint64_t bd = tc::umma_desc_sw128(a_addr + kA);
#pragma unroll
            for (int k = 0; k < BK / 32; ++k)
              umma_i8<false>(d, ad + 2 * k, bd + 2 * k, idesc, kb > 0 || k > 0 ? 1u : 0u);
            tc::umma_commit(&ctl->empty[s]);
          }
          __syncwarp();
          turn.next(p.stages);
        }
        if (ok && issues) tc::umma_commit(&ctl->tmem_full[b]);
        __syncwarp();
      }
      if (!ok && lane == 0) raise_fault(ctl, fault);
      if (issues) tc::umma_commit(&ctl->drain);
      tc::mbar_wait(&ctl->drain, 0, kWaitLimitNs, nullptr);
    }
  } else {
    // ---- epilogue: warp w drains row quarter w % 4, tokens 8 (w / 4) .. +7 of each pass; then
    // each warp sums the slices of two tokens, a channel a lane
    const int q = warp % 4, tok8 = (warp / 4) * 8;
    int n = 0;
    for (int t = blockIdx.x; t < p.tiles; t += gridDim.x, ++n) {
      const int b = n & 1, use = n >> 1;
      const int ch = t * kSliceCh + lane;
      const bool valid = ch < j.channels;
      const float sc = valid ? j.channel_scales[ch] : 0.f;
      const float sc2 = SILU && valid ? j.channel_scales[j.channels + ch] : 0.f;
      const float bias =
          !SILU && j.bias && valid ? Traits<T>::to_f(static_cast<const T*>(j.bias)[ch]) : 0.f;
      float st[kSliceTok / EPI_WARPS];  // the next pass's token scales
#pragma unroll
      for (int e = 0; e < kSliceTok / EPI_WARPS; ++e)
        st[e] = j.token_scales[min(warp + e * EPI_WARPS, j.tokens - 1)];
      bool ready =
          tc::mbar_wait(&ctl->tmem_full[b], (uint32_t)use & 1u, kWaitLimitNs, &ctl->abort);
      ready = epi_all(ready);
      if (!ready) {
        raise_fault(ctl, fault);
        break;
      }
      tc::tc_fence_after();
      const uint32_t acc = tmem + (uint32_t)(b * cols + (q % SL) * p.tc) + ((uint32_t)(q * 32) << 16);
#pragma unroll 1
      for (int tok0 = 0; tok0 < j.tokens; tok0 += kSliceTok) {
        if (tok0 + tok8 < p.tc) {
          uint32_t r[8];
          tmem_ld8(acc + (uint32_t)(tok0 + tok8), r);
          tc::tmem_wait_ld(r);
#pragma unroll
          for (int e = 0; e < 8; ++e) sums[(q * kSliceTok + tok8 + e) * kSliceCh + lane] = (int)r[e];
        }
        if (tok0 + kSliceTok >= j.tokens) {  // drained: the next tile's products may come
          tc::tc_fence_before();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(&ctl->tmem_empty[b]);
        }
        epi_sync();
#pragma unroll
        for (int e = 0; e < kSliceTok / EPI_WARPS; ++e) {
          const int i = warp + e * EPI_WARPS, tok = tok0 + i;
          if (tok < j.tokens && valid) {
            int v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = sums[(k * kSliceTok + i) * kSliceCh + lane];
            float y;
            if (SILU)
              y = silu_mul<T>((float)(v[0] + v[1]) * st[e] * sc, (float)(v[2] + v[3]) * st[e] * sc2);
            else
              y = (float)(v[0] + v[1] + v[2] + v[3]) * st[e] * sc + bias;
            if (j.add) y += Traits<T>::to_f(static_cast<const T*>(j.add)[tok * j.add_stride + ch]);
            static_cast<T*>(j.out)[tok * j.out_stride + ch] = Traits<T>::from_f(y);
          }
          st[e] = j.token_scales[min(tok + kSliceTok, j.tokens - 1)];
        }
        epi_sync();
      }
    }
  }

  tc::tc_fence_before();
  __syncthreads();
  if (warp == 0) tc::tmem_dealloc(tmem, (uint32_t)p.tmem_cols);
}

// ------------------------------------------------------- a middling number --
// 128 channels (64 gates and their 64 ups with SiLU) in the accumulator's rows and
// up to 128 tokens in its columns, K cut over the CTAs of a cluster: each works out
// a partial tile, puts it into its shared memory, and then sums its share of the
// tokens over the cluster's shared memories.  So the tile is large enough not to
// read the operands from L2 many times over, there are CTAs for all SMs, and the
// joining costs two cluster barriers.  Which CTA sums what is fixed, and sums of
// integers are exact.
constexpr int kMidRing = 98304;
constexpr int kMidAhead = 16;  // K blocks that are pulled into L2 before the wait
constexpr int kMidRest = 1024 + 256;
constexpr int kMidTok = 128;  // of a tile, at most

struct MidTiling {
  int bt, stages, ring, tmem_cols, tok_tiles, cut;  // tokens a tile; CTAs of a cluster
};

// 16 bytes of the shared memory of the cluster's CTA `rank`, at this CTA's address p.
__device__ __forceinline__ int4 ld_cluster(const int32_t* p, uint32_t rank) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(tc::map_to_rank(p, rank))
               : "memory");
  return v;
}

template <typename T, bool SILU>
__global__ void __launch_bounds__(THREADS, 2)
    int8_mid_kernel(const __grid_constant__ CUtensorMap tm_w,
                    const __grid_constant__ CUtensorMap tm_x, const GemmJob j, const MidTiling p,
                    int32_t* fault) {
  constexpr int kA = BM * BK, kOut = SILU ? BM / 2 : BM;  // channels of a tile
  extern __shared__ uint8_t smem_raw[];
  uint8_t* tiles = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  int32_t* part = reinterpret_cast<int32_t*>(tiles);  // [token][row], over the ring
  Ctl* ctl = reinterpret_cast<Ctl*>(tiles + p.ring);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sb = kA + p.bt * BK;  // bytes of a stage
  const int rank = (int)tc::cluster_rank();
  const int tile = (int)blockIdx.x / p.cut;
  const int n0 = tile / p.tok_tiles * kOut, t0 = tile % p.tok_tiles * p.bt;
  const int kb0 = (int)((int64_t)rank * j.k_blocks / p.cut);
  const int kb1 = (int)((int64_t)(rank + 1) * j.k_blocks / p.cut);

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      tc::mbar_init(&ctl->full[s], 1);
      tc::mbar_init(&ctl->empty[s], 1);
    }
    tc::mbar_init(&ctl->tmem_full[0], 1);
    ctl->abort = 0;
    tc::fence_barrier_init();
  }
  if (warp == EPI_WARPS && lane == 0) {
    tc::tma_prefetch_desc(&tm_w);
    tc::tma_prefetch_desc(&tm_x);
    // L2 is the point of coherence: what an earlier kernel still writes to the weight is read from
    // there after the wait
    for (int kb = kb0; kb < min(kb1, kb0 + kMidAhead); ++kb) {
      prefetch_box(&tm_w, kb * BK, n0);
      if (SILU) prefetch_box(&tm_w, kb * BK, j.channels + n0);
    }
  }
  if (warp == 0) tc::tmem_alloc(&ctl->tmem, (uint32_t)p.tmem_cols);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = ctl->tmem;
  pdl_launch_dependents();
  pdl_wait();

  if (warp == EPI_WARPS) {
    // ---- TMA producer: the whole warp walks, one lane issues ------------------
    {
      const bool issues = elect_one();
      bool ok = true;
      Turn turn;
      int i = 0;
      for (int kb = kb0; kb < kb1; ++kb, ++i) {
        const int s = turn.s;
        if (i >= p.stages && !ring_wait(&ctl->empty[s], turn.phase ^ 1u, ctl)) {
          ok = false;
          break;
        }
        if (issues) {
          uint8_t* a = tiles + s * sb;
          tc::mbar_arrive_expect_tx(&ctl->full[s], (uint32_t)sb);
          tc::tma_load_2d(a, &tm_w, kb * BK, n0, &ctl->full[s]);
          if (SILU) tc::tma_load_2d(a + kA / 2, &tm_w, kb * BK, j.channels + n0, &ctl->full[s]);
          tc::tma_load_2d(a + kA, &tm_x, kb * BK, t0, &ctl->full[s]);
        }
        __syncwarp();
        turn.next(p.stages);
      }
      if (!ok && lane == 0) raise_fault(ctl, fault);
      for (int q = i > p.stages ? i - p.stages : 0; q < i; ++q)
        tc::mbar_wait(&ctl->full[q % p.stages], (uint32_t)(q / p.stages) & 1u, kWaitLimitNs, nullptr);
    }
  } else if (warp == EPI_WARPS + 1) {
    // ---- MMA issuer ---------------------------------------------------------
    {
      const bool issues = elect_one();
      const uint32_t idesc = idesc_i8(BM, p.bt);
      bool ok = true;
      Turn turn;
      for (int kb = kb0; kb < kb1; ++kb) {
        const int s = turn.s;
        if (!ring_wait(&ctl->full[s], turn.phase, ctl)) {
          ok = false;
          break;
        }
        tc::tc_fence_after();
        if (issues) {
          const uint32_t a_addr = tc::smem_u32(tiles + s * sb);
          const uint64_t ad = tc::umma_desc_sw128(a_addr);
          const uint64_t bd = tc::umma_desc_sw128(a_addr + kA);
#pragma unroll
          for (int k = 0; k < BK / 32; ++k)
            umma_i8<false>(tmem, ad + 2 * k, bd + 2 * k, idesc, kb > kb0 || k > 0 ? 1u : 0u);
          tc::umma_commit(&ctl->empty[s]);
        }
        __syncwarp();
        turn.next(p.stages);
      }
      if (!ok && lane == 0) raise_fault(ctl, fault);
      // the last commit follows all products, whether or not all were issued
      if (issues) tc::umma_commit(&ctl->tmem_full[0]);
      tc::mbar_wait(&ctl->tmem_full[0], 0, kWaitLimitNs, nullptr);
    }
  } else {
    // ---- the partial tile goes to shared memory: warp w row quarter w % 4, half w / 4 of the tokens
    const int row = (warp % 4) * 32 + lane, c0 = (warp / 4) * (p.bt / 2);
    const bool ready = tc::mbar_wait(&ctl->tmem_full[0], 0, kWaitLimitNs, &ctl->abort);
    // all eight take one way: the ring is written over only when every product has read it
    if (epi_all(ready)) {
      tc::tc_fence_after();
      const uint32_t acc = tmem + ((uint32_t)(warp % 4 * 32) << 16);
#pragma unroll 1
      for (int c = c0; c < c0 + p.bt / 2 && t0 + c < j.tokens; c += 8) {
        uint32_t r[8];
        tmem_ld8(acc + (uint32_t)c, r);
        tc::tmem_wait_ld(r);
#pragma unroll
        for (int e = 0; e < 8; ++e) part[(c + e) * BM + row] = (int)r[e];
      }
    } else {
      raise_fault(ctl, fault);
    }
  }
  tc::tc_fence_before();
  __syncwarp();
  tc::cluster_sync();

  // ---- a warp a token (two with SiLU), four channels a lane, summed over the cluster -----------
  {
    constexpr int kLanes = kOut / 4, kEach = 32 / kLanes;  // of a token; tokens of a warp
    const int ch = n0 + (lane % kLanes) * 4;
    const bool four = ch + 4 <= j.channels;
    float sc[4], sc2[4], bias[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int n = min(ch + e, j.channels - 1);
      sc[e] = __ldg(j.channel_scales + n);
      sc2[e] = SILU ? __ldg(j.channel_scales + j.channels + n) : 0.f;
      bias[e] = !SILU && j.bias ? Traits<T>::to_f(static_cast<const T*>(j.bias)[n]) : 0.f;
    }
    const int end = min(p.bt, j.tokens - t0);
    for (int c = rank + (warp * kEach + lane / kLanes) * p.cut; c < end;
         c += (THREADS / 32) * kEach * p.cut) {
      int4 v = make_int4(0, 0, 0, 0), u = v;
      const int32_t* at = part + c * BM + (lane % kLanes) * 4;
#pragma unroll 4
      for (int k = 0; k < p.cut; ++k) {
        const int4 x = ld_cluster(at, (uint32_t)k);
        v.x += x.x;
        v.y += x.y;
        v.z += x.z;
        v.w += x.w;
        if (SILU) {
          const int4 z = ld_cluster(at + BM / 2, (uint32_t)k);
          u.x += z.x;
          u.y += z.y;
          u.z += z.z;
          u.w += z.w;
        }
      }
      const int64_t t = t0 + c;
      const float st = j.token_scales[t];
      const int g[4] = {v.x, v.y, v.z, v.w}, h[4] = {u.x, u.y, u.z, u.w};
      float y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        y[e] = (float)g[e] * st * sc[e] + bias[e];
        if (SILU) y[e] = silu_mul<T>(y[e], (float)h[e] * st * sc2[e]);
      }
      put_four<T>(j, t, ch, four, y);
    }
  }
  // no CTA leaves while another reads its shared memory
  __syncwarp();
  tc::cluster_sync();
  if (warp == 0) tc::tmem_dealloc(tmem, (uint32_t)p.tmem_cols);
}

// ------------------------------------------------------------ any rows --
// Any K, stride and alignment: 32 tokens x 32 channels a CTA, 256 bytes of K at a
// time through shared memory, a 16 x 8 x 32 matrix instruction's tile a warp.  A
// row is read in the aligned words that hold its bytes, shifted together (77
// tokens, K 1111, 1003 channels: byte by byte 54 us).  The next step's words are
// under way while this one's products are formed; the latency of those few steps
// bounds it.
constexpr int kDotK = 256, kDotTok = 32, kDotCh = 32, kDotPitch = kDotK + 16;
constexpr int kDotThreads = 256;

// 16 bytes at `at` of a row of k bytes, zero past its end.
__device__ __forceinline__ uint4 row_bytes(const int8_t* row, int at, int k) {
  uint32_t v[4] = {};
  if (at < k) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(row + at), end = reinterpret_cast<uintptr_t>(row + k);
    const uint32_t* words = reinterpret_cast<const uint32_t*>(p & ~static_cast<uintptr_t>(3));
    const int shift = (int)(p & 3) * 8;
    uint32_t w[5];
#pragma unroll
    for (int i = 0; i < 5; ++i)  // no word without a byte of the row
      w[i] = reinterpret_cast<uintptr_t>(words + i) < end ? words[i] : 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = __funnelshift_r(w[i], w[i + 1], shift);
      const int left = k - at - 4 * i;  // bytes of this word in the row
      if (left < 4) v[i] = left <= 0 ? 0u : v[i] & ((1u << (8 * left)) - 1u);
    }
  }
  return make_uint4(v[0], v[1], v[2], v[3]);
}

template <typename T, bool SILU>
__global__ void __launch_bounds__(kDotThreads)
    int8_dot_kernel(const int8_t* codes, int64_t codes_stride, const int8_t* weight,
                    int64_t weight_stride, int k, const GemmJob j) {
  constexpr int NW = SILU ? 2 : 1, kRows = kDotTok + NW * kDotCh;
  constexpr int kEach = kRows * (kDotK / 16) / kDotThreads;
  static_assert(kEach * kDotThreads == kRows * (kDotK / 16), "");
  __shared__ __align__(16) int8_t rows[kRows][kDotPitch];  // tokens, then channels
  const int64_t t0 = (int64_t)blockIdx.x * kDotTok;
  const int n0 = (int)blockIdx.y * kDotCh;
  const int warp = threadIdx.x >> 5, g = (threadIdx.x & 31) >> 2, c = threadIdx.x & 3;
  const int wt = warp / 4 * 16, wc = warp % 4 * 8;  // the warp's tokens and channels
  pdl_launch_dependents();
  pdl_wait();
  uint4 next[kEach];
  auto fetch = [&](int k0) {
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int i = threadIdx.x + e * kDotThreads, r = i / (kDotK / 16), at = i % (kDotK / 16) * 16;
      next[e] = make_uint4(0, 0, 0, 0);
      if (r < kDotTok) {
        if (t0 + r < j.tokens) next[e] = row_bytes(codes + (t0 + r) * codes_stride, k0 + at, k);
      } else {
        const int h = (r - kDotTok) / kDotCh, n = n0 + (r - kDotTok) % kDotCh;
        if (n < j.channels)
          next[e] = row_bytes(weight + ((int64_t)h * j.channels + n) * weight_stride, k0 + at, k);
      }
    }
  };
  int acc[NW][4] = {};
  fetch(0);
  for (int k0 = 0; k0 < k; k0 += kDotK) {
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int i = threadIdx.x + e * kDotThreads, r = i / (kDotK / 16), at = i % (kDotK / 16) * 16;
      *reinterpret_cast<uint4*>(&rows[r][at]) = next[e];
    }
    __syncthreads();
    if (k0 + kDotK < k) fetch(k0 + kDotK);
#pragma unroll
    for (int s = 0; s < kDotK; s += 32) {
      auto word = [&](int r, int at) { return *reinterpret_cast<const uint32_t*>(&rows[r][at + 4 * c]); };
      const uint32_t a0 = word(wt + g, s), a1 = word(wt + g + 8, s), a2 = word(wt + g, s + 16),
                     a3 = word(wt + g + 8, s + 16);
#pragma unroll
      for (int h = 0; h < NW; ++h) {
        const int r = kDotTok + h * kDotCh + wc + g;
        asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
            "{%0,%1,%2,%3};"
            : "+r"(acc[h][0]), "+r"(acc[h][1]), "+r"(acc[h][2]), "+r"(acc[h][3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(word(r, s)), "r"(word(r, s + 16)));
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int64_t t = t0 + wt + g + e / 2 * 8;
    const int n = n0 + wc + 2 * c + e % 2;
    if (t >= j.tokens || n >= j.channels) continue;
    const float st = j.token_scales[t];
    float y = (float)acc[0][e] * st * j.channel_scales[n];
    if (SILU)
      y = silu_mul<T>(y, (float)acc[NW - 1][e] * st * j.channel_scales[j.channels + n]);
    else if (j.bias)
      y += Traits<T>::to_f(static_cast<const T*>(j.bias)[n]);
    if (j.add) y += Traits<T>::to_f(static_cast<const T*>(j.add)[t * j.add_stride + n]);
    static_cast<T*>(j.out)[t * j.out_stride + n] = Traits<T>::from_f(y);
  }
}

// -------------------------------------------------------------- host side --
struct Call {
  const int8_t *codes, *weight;
  int64_t codes_stride, weight_stride, tokens, k, channels;
  bool silu;
  int32_t* fault;
  int dtype, device;
  cudaStream_t stream;
  const char* name;
};

constexpr int64_t kSliceTokens = 32;  // up to here the slice kernel
constexpr int64_t kMidTokens = 128;   // up to here the cluster kernel, above by rows_plan

// Tiles for the rows kernel: 128, 192 or 256 channels, whichever takes least by what a round of tiles
// over the pairs costs (B200, ns a K block, and us for a call's start and end):
//   128: 195, 6.8;  192: 275, 8.0;  256: 295, 9.1
// (512 tokens, K 4096: 6144 channels 19.2, 17.5, 19.3 us; 4096 channels 13.4, 16.7, 18.5.)
// A last round that would leave half of the pairs idle takes its tiles of 256 in halves, at 190 ns a
// K block (512 tokens, K 4096: gate and up of 14336, 2 tiles of 224 left, 47.9 us against 50.1; 20000
// channels, 10 of 158 left, 37.0 against 39.0).
struct RowsPlan {
  Tiling t;
  int pairs;
};
inline RowsPlan rows_plan(int64_t tokens, int64_t channels, int k_blocks, bool silu, int sms) {
  static constexpr struct {
    int bn;
    double block, fixed;
  } kinds[] = {{128, 0.195, 6.8}, {192, 0.275, 8.0}, {256, 0.295, 9.1}};
  RowsPlan best = {};
  double least = 0;
  const int pairs = std::max(1, sms / 2);
  for (const auto& kind : kinds) {
    const int64_t m = ceil_div(tokens, 2 * BM), n = ceil_div(channels, silu ? kind.bn / 2 : kind.bn);
    const int64_t last = m * n % pairs;  // tiles of the last round
    const bool halves = kind.bn == 256 && m * n > pairs && 2 * last <= pairs;
    const double cost = kind.fixed + k_blocks * ((double)(m * n / pairs) * kind.block +
                                                 (last == 0 ? 0. : halves ? 0.19 : kind.block));
    if (best.pairs != 0 && cost >= least) continue;
    least = cost;
    best.t.bn = kind.bn;
    best.t.m_tiles = (int)m;
    best.t.n_tiles = (int)n;
    best.t.whole = halves ? m * n - last : m * n;
    best.pairs = (int)std::min<int64_t>(m * n, pairs);
  }
  // two K blocks a stage halve what a stage costs beside its bytes (128 channels: 270 -> 195 ns);
  // at 256 the products take longer than that anyway, and more stages are better
  best.t.sub = best.t.bn == 256 ? 1 : 2;
  best.t.stages = std::min(MAX_STAGES, kRingBytes / (best.t.sub * (BM + best.t.bn / 2) * BK));
  return best;
}

// Boxes of `box` rows of a K block, or (deep, where K is whole blocks) of `blocks`
// K blocks: the third axis steps by a block within the row.
int make_map(CUtensorMap* map, const int8_t* base, int64_t rows, int64_t k, int64_t stride, int box,
             bool deep, int blocks, const char* name) {
  tc::EncodeTiledFn enc = tc::encode_tiled();
  if (!enc) return fail(PACE_ERR_CUDA, "%s: cuTensorMapEncodeTiled unavailable", name);
  const cuuint64_t dims[3] = {(cuuint64_t)(deep ? BK : k), (cuuint64_t)rows, (cuuint64_t)(k / BK)};
  const cuuint64_t strides[2] = {(cuuint64_t)stride, (cuuint64_t)BK};
  const cuuint32_t boxes[3] = {(cuuint32_t)BK, (cuuint32_t)box, (cuuint32_t)blocks};
  const cuuint32_t steps[3] = {1, 1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, deep ? 3 : 2, const_cast<int8_t*>(base),
                         dims, strides, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(PACE_ERR_INVALID_ARGUMENT, "%s: tensor map rejected (CUresult %d)", name, (int)r);
  return PACE_OK;
}

inline int64_t weight_rows(const Call& c) { return c.silu ? 2 * c.channels : c.channels; }

template <typename T, bool SILU>
int launch_slices(const Call& c, const GemmJob& j) {
  constexpr int SL = SILU ? 2 : 4;
  SliceTiling p;
  p.tc = (int)ceil_div(c.tokens, 8) * 8;
  p.tiles = (int)ceil_div(c.channels, kSliceCh);
  const int stage = BM * BK + SL * p.tc * BK;
  p.slice_blocks = (int)ceil_div(j.k_blocks, SL);
  // With a tile for each SM at most, and more blocks than two turns of the ring, one CTA an SM takes
  // the whole shared memory (a token, K 14336, 4096 channels: 12.3 us against 14.4); a short K has
  // no use for it (K 4096: 5.6 against 5.5)
  p.stages = kSliceRing / stage;
  if (p.tiles <= sm_count(c.device) && p.slice_blocks > 2 * p.stages) p.stages = kRingBytes / stage;
  p.stages = std::min(MAX_STAGES, p.stages);
  p.ring = p.stages * stage;
  p.tmem_cols = 32;  // two accumulators
  while (p.tmem_cols < 2 * SL * p.tc) p.tmem_cols *= 2;
  CUtensorMap w, x;
  int rc = make_map(&w, c.weight, weight_rows(c), c.k, c.weight_stride, kSliceCh, j.deep, SL, c.name);
  if (rc == PACE_OK)
    rc = make_map(&x, c.codes, c.tokens, c.k, c.codes_stride, p.tc, j.deep, SL, c.name);
  if (rc != PACE_OK) return rc;
  auto kernel = int8_slice_kernel<T, SILU>;
  cudaError_t err = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), c.device, kRingBytes + kSliceRest);
  if (err != cudaSuccess) return cuda_fail(err, c.name);
  const int grid = std::min(p.tiles, 2 * sm_count(c.device));
  err = launch(kernel, dim3((unsigned)grid), dim3(THREADS), p.ring + kSliceRest, c.stream, w, x, j, p, c.fault);
  return err == cudaSuccess ? PACE_OK : cuda_fail(err, c.name);
}

template <typename T, bool SILU>
int launch_mid(const Call& c, const GemmJob& j) {
  MidTiling p;
  p.tok_tiles = (int)ceil_div(c.tokens, kMidTok);
  p.bt = (int)ceil_div(ceil_div(c.tokens, p.tok_tiles), 16) * 16;
  p.tmem_cols = 32;
  while (p.tmem_cols < p.bt) p.tmem_cols *= 2;
  const int tiles = (int)ceil_div(c.channels, SILU ? BM / 2 : BM) * p.tok_tiles;
  // K is cut for two CTAs an SM, with 8 K blocks each at least (4096 x 4096, 64 tokens: 8 blocks 8.7
  // us, 4 blocks 9.6), in clusters of a power of two, which find room on the SMs (48 tiles of 128
  // channels, 64 tokens: clusters of 4 10.1 us, of 6 17.1)
  const int sms = sm_count(c.device), stage = BM * BK + p.bt * BK;
  auto cut_for = [&](int ctas) {
    int cut = 1;
    while (cut < 8 && tiles * cut * 2 <= ctas && j.k_blocks / (cut * 2) >= 8) cut *= 2;
    return cut;
  };
  p.cut = cut_for(2 * sms);
  p.ring = kMidRing;
  // or for one CTA, with a ring twice as long, where that leaves few SMs without any and its part
  // of K fills the ring (4096 channels, K 14336, 64 / 128 tokens: 15.8 / 17.8 us against 16.4 /
  // 19.9; 6144 channels, K 4096, 96 CTAs: 13.4 against 12.7)
  const int one = cut_for(sms);
  if (tiles * one <= sms && 5 * tiles * one >= 4 * sms && j.k_blocks / one * stage > kRingBytes) {
    p.cut = one;
    p.ring = kRingBytes;
  }
  p.stages = std::min(MAX_STAGES, p.ring / stage);
  CUtensorMap w, x;
  int rc = make_map(&w, c.weight, weight_rows(c), c.k, c.weight_stride, SILU ? BM / 2 : BM, false, 1,
                    c.name);
  if (rc == PACE_OK)
    rc = make_map(&x, c.codes, c.tokens, c.k, c.codes_stride, p.bt, false, 1, c.name);
  if (rc != PACE_OK) return rc;
  auto kernel = int8_mid_kernel<T, SILU>;
  cudaError_t err = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), c.device, kRingBytes + kMidRest);
  if (err != cudaSuccess) return cuda_fail(err, c.name);
  err = launch_clusters(kernel, p.cut, dim3((unsigned)(tiles * p.cut)), dim3(THREADS), p.ring + kMidRest,
                        c.stream, w, x, j, p, c.fault);
  return err == cudaSuccess ? PACE_OK : cuda_fail(err, c.name);
}

template <typename T, bool SILU>
int launch_rows(const Call& c, const GemmJob& j, const RowsPlan& p) {
  CUtensorMap a, b, half;
  int rc = make_map(&a, c.codes, c.tokens, c.k, c.codes_stride, BM, j.deep, p.t.sub, c.name);
  if (rc == PACE_OK)
    rc = make_map(&b, c.weight, weight_rows(c), c.k, c.weight_stride, p.t.bn / 2, j.deep, p.t.sub,
                  c.name);
  half = b;
  if (rc == PACE_OK && p.t.whole < (int64_t)p.t.m_tiles * p.t.n_tiles)
    rc = make_map(&half, c.weight, weight_rows(c), c.k, c.weight_stride, p.t.bn / 4, j.deep, p.t.sub,
                  c.name);
  if (rc != PACE_OK) return rc;
  auto kernel = int8_gemm_kernel<T, SILU>;
  cudaError_t err = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), c.device, kSmem + kTurn);
  if (err != cudaSuccess) return cuda_fail(err, c.name);
  err = launch_pairs(kernel, dim3((unsigned)(2 * p.pairs)), dim3(THREADS),
                     j.vec ? kSmem : kSmem + kTurn, c.stream, a, b, half,
                     j, p.t, c.fault);
  return err == cudaSuccess ? PACE_OK : cuda_fail(err, c.name);
}

template <typename T, bool SILU>
int launch_tensor(const Call& c, const GemmJob& j) {
  if (c.tokens <= kSliceTokens) return launch_slices<T, SILU>(c, j);
  // more tokens go to the cluster kernel too where whole tiles would leave half of the SMs idle
  // (256 tokens, K 14336, 4096 channels: 22 us against 28)
  const int sms = sm_count(c.device);
  const RowsPlan p = rows_plan(c.tokens, c.channels, j.k_blocks, SILU, sms);
  return c.tokens <= kMidTokens || p.pairs <= sms / 4 ? launch_mid<T, SILU>(c, j)
                                                      : launch_rows<T, SILU>(c, j, p);
}

// Whether TMA takes both operands.
inline bool for_tma(const Call& c) {
  return c.codes_stride % 16 == 0 && c.weight_stride % 16 == 0 && aligned16(c.codes) &&
         aligned16(c.weight);
}

template <typename T>
int run_typed(const Call& c, GemmJob j) {
  constexpr int V = Traits<T>::kVec;
  j.vec = aligned16(j.out) && j.out_stride % V == 0 &&
          (!j.add || (aligned16(j.add) && j.add_stride % V == 0));
  j.scales_vec = aligned16(j.channel_scales) && (!c.silu || c.channels % 4 == 0);
  j.k_blocks = (int)ceil_div(c.k, BK);
  j.deep = c.k % BK == 0;
  if (for_tma(c)) return c.silu ? launch_tensor<T, true>(c, j) : launch_tensor<T, false>(c, j);
  const dim3 grid((unsigned)ceil_div(c.tokens, kDotTok), (unsigned)ceil_div(c.channels, kDotCh));
  if (grid.y > 65535)
    return fail(PACE_ERR_TOO_LARGE, "%s: over 2097120 channels of rows that are not 16-byte aligned",
                c.name);
  const cudaError_t err =
      c.silu ? launch(int8_dot_kernel<T, true>, grid, dim3(kDotThreads), 0, c.stream, c.codes,
                      c.codes_stride, c.weight, c.weight_stride, (int)c.k, j)
             : launch(int8_dot_kernel<T, false>, grid, dim3(kDotThreads), 0, c.stream, c.codes,
                      c.codes_stride, c.weight, c.weight_stride, (int)c.k, j);
  return err == cudaSuccess ? PACE_OK : cuda_fail(err, c.name);
}

int run_int8(Call c, GemmJob j) {
  if (c.tokens < 0 || c.tokens > kMaxRows || c.channels <= 0 || c.channels > kMaxRows || c.k <= 0)
    return fail(PACE_ERR_INVALID_ARGUMENT, "%s: bad shape", c.name);
  if (c.k > kMaxK)
    return fail(PACE_ERR_TOO_LARGE, "%s: k %lld: sums of more than %lld products may not fit 32 bits",
                c.name, (long long)c.k, (long long)kMaxK);
  if (c.codes_stride < c.k || c.weight_stride < c.k || j.out_stride < c.channels ||
      (j.add && j.add_stride < c.channels))
    return fail(PACE_ERR_INVALID_ARGUMENT, "%s: row stride smaller than the row", c.name);
  if (c.tokens == 0) return PACE_OK;
  if (!c.codes || !c.weight || !j.out || !j.token_scales || !j.channel_scales)
    return fail(PACE_ERR_INVALID_ARGUMENT, "%s: null pointer", c.name);
  StreamDeviceGuard guard(c.stream);
  c.device = guard.device();
  if (c.tokens == 1) c.codes_stride = ceil_div(c.k, 16) * 16;  // of one row it says nothing
  j.tokens = (int)c.tokens;
  j.channels = (int)c.channels;
  return PACE_DISPATCH_FLOAT(c.dtype, c.name, [&] { return run_typed<scalar_t>(c, j); });
}

}  // namespace
}  // namespace pace

extern "C" int pace_int8_linear(void* out, const int8_t* codes, const float* token_scales,
                                const int8_t* weight, const float* channel_scales,
                                const void* bias, const void* residual, int64_t num_tokens,
                                int64_t out_features, int64_t k, int64_t codes_row_stride,
                                int64_t weight_row_stride, int64_t out_row_stride,
                                int64_t residual_row_stride, int dtype, int32_t* fault_flags,
                                cudaStream_t stream) {
  pace::GemmJob j = {};
  j.out = out;
  j.add = residual;
  j.bias = bias;
  j.token_scales = token_scales;
  j.channel_scales = channel_scales;
  j.out_stride = out_row_stride;
  j.add_stride = residual_row_stride;
  return pace::run_int8({codes, weight, codes_row_stride, weight_row_stride, num_tokens, k,
                         out_features, false, fault_flags, dtype, 0, stream, "int8_linear"},
                        j);
}

extern "C" int pace_int8_gate_up_silu(void* out, const int8_t* codes, const float* token_scales,
                                      const int8_t* weight, const float* channel_scales,
                                      int64_t num_tokens, int64_t intermediate_size, int64_t k,
                                      int64_t codes_row_stride, int64_t weight_row_stride,
                                      int64_t out_row_stride, int dtype, int32_t* fault_flags,
                                      cudaStream_t stream) {
  pace::GemmJob j = {};
  j.out = out;
  j.token_scales = token_scales;
  j.channel_scales = channel_scales;
  j.out_stride = out_row_stride;
  return pace::run_int8({codes, weight, codes_row_stride, weight_row_stride, num_tokens, k,
                         intermediate_size, true, fault_flags, dtype, 0, stream, "int8_gate_up_silu"},
                        j);
}
