// Products of 8-bit integers with a scale for each token and each output
// channel, for sm_100a: the projections of a decoder layer with 8-bit weights.
//
//   y_tn = (sum_k c_tk w_nk) * s_t * s_n  (+ bias_n) (+ residual_tn)
//   gate_up_silu:  silu(y_tn) * y_t(I + n),   weight [2 I, K]
//
// The sum is int32, so it is exact and the same in every order of its terms (K is
// at most 131071, where 128 * 128 * K still fits); the rest is fp32, rounded once.
//
// One kernel (int8_gemm_kernel): TMA fills a ring of 128-byte K blocks (128-byte
// swizzle), one thread issues tcgen05.mma.kind::i8 into one of two TMEM
// accumulators, and eight warps drain the other through the scales.  Two ways
// round:
//  * tokens in the accumulator's rows (its lanes), channels in its columns: 256
//    tokens on a CTA pair (cta_group::2) or 128 on one CTA, by 256 channels;
//  * few tokens: channels in the rows, tokens in 16 to 64 columns, so that a
//    decode batch's tile is not padding but the weight, and what is drained is
//    small.  There the weight's bytes bound it.
// Tiles that do not fill the SMs evenly are cut over K (stream-K): workers leave
// int32 partial sums in the workspace, and the last to arrive at a tile adds them
// up.  No CTA waits for another, and the result does not depend on who is last.
//
// What TMA cannot take (K, a row stride or an address that is no multiple of 16
// bytes) runs on the CUDA cores (int8_dot_kernel).
#include <algorithm>

#include "tcgen05.cuh"

namespace pace {
namespace {

constexpr int BK = 128;  // bytes of K per stage: one swizzle atom
constexpr int BM = 128;
constexpr int EPI_WARPS = 8;
constexpr int THREADS = (EPI_WARPS + 2) * 32;
constexpr int MAX_STAGES = 10;
constexpr int kRingBytes = 196608;  // at most
constexpr int kEpiBarrier = 1;
constexpr uint64_t kWaitLimitNs = 1000000000ull;  // 1 s per wait
constexpr int32_t kFaultTimeout = 1 << 30;
constexpr int64_t kMaxK = 131071;
// The workspace: arrival counters of the tiles that are cut, then the partial sums.
constexpr int64_t kCounterBytes = 4096;

struct Ctl {
  uint64_t full[MAX_STAGES];
  uint64_t empty[MAX_STAGES];
  uint64_t tmem_full[2];
  uint64_t tmem_empty[2];
  uint64_t drain;
  uint32_t tmem;
  int abort;
  int last;
};
static_assert(sizeof(Ctl) <= 256, "");

struct GemmJob {
  void* out;
  const void* add;   // residual, or null
  const void* bias;  // or null
  const float *token_scales, *channel_scales;
  int64_t out_stride, add_stride;
  int tokens, channels;  // channels: output columns (half the weight's rows with SiLU)
  int k_blocks, m_tiles, n_tiles;
  int vec;  // out (and add) take 16-byte accesses
};

// TOK_ROWS: tokens in the accumulator's rows.  SILU: each tile has a gate and an
// up part: the two halves of its columns (TOK_ROWS), or two accumulators.
template <int BN_, bool PAIR_, bool TOK_ROWS_, bool SILU_>
struct Shape {
  static constexpr int BN = BN_;
  static constexpr bool PAIR = PAIR_, TOK_ROWS = TOK_ROWS_, SILU = SILU_;
  static constexpr int NACC = SILU && !TOK_ROWS ? 2 : 1;
  static constexpr int kA = NACC * BM * BK;            // bytes per CTA and stage
  static constexpr int kB = (PAIR ? BN / 2 : BN) * BK;
  static constexpr int kStage = kA + kB;
  static constexpr int kStages = kRingBytes / kStage < MAX_STAGES ? kRingBytes / kStage : MAX_STAGES;
  static constexpr int kSmem = kStages * kStage + 1024 + 256;
  static constexpr int kRows = PAIR ? 2 * BM : BM;     // of a tile
  static constexpr int kCols = NACC * BN;              // accumulator columns
  static constexpr int kTmem = 2 * kCols < 32 ? 32 : 2 * kCols;
  static constexpr int kOutCols = SILU && TOK_ROWS ? BN / 2 : BN;  // output columns of a tile
  static constexpr int kHalf = kOutCols / 2;           // of one of the two warps of a lane quarter
  static constexpr int CH = kHalf < 16 ? kHalf : 16;   // columns drained at a time
  static constexpr int kSlot = kCols * BM;             // int32 of a partial tile
  static_assert(kTmem <= 512 && (kTmem & (kTmem - 1)) == 0 && CH % 8 == 0, "");
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

// N (8 or 16) consecutive columns of this thread's TMEM lane; valid after
// tc::tmem_wait_ld.
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&r)[16]) {
  tc::tmem_ld16(taddr, r);
}
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7])
      : "r"(taddr)
      : "memory");
}

// Split of the K blocks of the tiles [t_stop, ...) over the first `workers` workers.
struct Split {
  int64_t units;
  int workers, k_blocks;
  __device__ __forceinline__ int64_t start(int w) const { return (int64_t)w * units / workers; }
  __device__ __forceinline__ int owner(int64_t u) const {
    return (int)(((u + 1) * workers - 1) / units);
  }
};

// A worker's segments in order: whole tiles worker, worker + step, ... below
// t_stop, then its range of the units of the tiles from t_stop on.
struct Walk {
  int64_t t_next, t_stop, step;
  int64_t u, u_end;
  int k_blocks;
  __device__ __forceinline__ bool next(int64_t& t, int& kb0, int& kb1) {
    if (t_next < t_stop) {
      t = t_next;
      t_next += step;
      kb0 = 0;
      kb1 = k_blocks;
      return true;
    }
    if (u >= u_end) return false;
    const int64_t rt = u / k_blocks;
    t = t_stop + rt;
    kb0 = (int)(u - rt * k_blocks);
    kb1 = (int)min((int64_t)k_blocks, kb0 + (u_end - u));
    u += kb1 - kb0;
    return true;
  }
};

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

// 16-bit outputs take the approximate exponential and quotient, a few units of
// 2^-24 that their own rounding hides; float32 the library's.
template <typename T>
__device__ __forceinline__ float silu_mul(float g, float u) {
  if constexpr (sizeof(T) == 2) return __fdividef(g, 1.f + __expf(-g)) * u;
  return g / (1.f + expf(-g)) * u;
}

// Partial sums: [4 columns][lane][4], so that a warp's instruction moves 512
// contiguous bytes; through L2 only, since another SM reads them.
template <int CH>
__device__ __forceinline__ void store_partial(int32_t* slot, int col, int row,
                                              const uint32_t (&r)[CH]) {
#pragma unroll
  for (int q = 0; q < CH / 4; ++q)
    __stcg(reinterpret_cast<uint4*>(slot + ((int64_t)(col / 4 + q) * BM + row) * 4),
           make_uint4(r[4 * q], r[4 * q + 1], r[4 * q + 2], r[4 * q + 3]));
}
template <int CH>
__device__ __forceinline__ void add_partial(const int32_t* slot, int col, int row,
                                            uint32_t (&r)[CH]) {
#pragma unroll
  for (int q = 0; q < CH / 4; ++q) {
    const uint4 v =
        __ldcg(reinterpret_cast<const uint4*>(slot + ((int64_t)(col / 4 + q) * BM + row) * 4));
    r[4 * q] += v.x;
    r[4 * q + 1] += v.y;
    r[4 * q + 2] += v.z;
    r[4 * q + 3] += v.w;
  }
}

// CH consecutive channels n .. of one token: add, round, store.
template <typename T, int CH>
__device__ __forceinline__ void put_channels(const GemmJob& j, int64_t t, int n, float* y) {
  constexpr int V = Traits<T>::kVec;
  T* o = static_cast<T*>(j.out) + t * j.out_stride + n;
  const T* add = j.add ? static_cast<const T*>(j.add) + t * j.add_stride + n : nullptr;
  if (j.vec && n + CH <= j.channels) {
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

template <typename T, class S>
__global__ void __launch_bounds__(THREADS, 1)
    int8_gemm_kernel(const __grid_constant__ CUtensorMap tm_a,
                     const __grid_constant__ CUtensorMap tm_b, const GemmJob j, int split_workers,
                     int32_t* counters, int32_t* slots, int32_t* fault) {
  constexpr bool PAIR = S::PAIR, TOK_ROWS = S::TOK_ROWS, SILU = S::SILU;
  constexpr int BN = S::BN, NST = S::kStages, SB = S::kStage, CH = S::CH;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* tiles = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  Ctl* ctl = reinterpret_cast<Ctl*>(tiles + NST * SB);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cta = blockIdx.x;
  const uint32_t rank = PAIR ? tc::cluster_rank() : 0u;
  const int worker = PAIR ? cta >> 1 : cta;
  const int workers = PAIR ? (int)gridDim.x >> 1 : (int)gridDim.x;
  const int64_t n_all = (int64_t)j.m_tiles * j.n_tiles;
  const int64_t t_stop = n_all / workers * workers;
  Split sp;
  sp.units = (n_all - t_stop) * j.k_blocks;
  sp.workers = split_workers;
  sp.k_blocks = j.k_blocks;
  const bool splits = worker < split_workers;
  const Walk walk0{worker,
                   t_stop,
                   (int64_t)workers,
                   splits ? sp.start(worker) : 0,
                   splits ? sp.start(worker + 1) : 0,
                   j.k_blocks};

  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int s = 0; s < NST; ++s) {
      tc::mbar_init(&ctl->full[s], 1);
      tc::mbar_init(&ctl->empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      tc::mbar_init(&ctl->tmem_full[b], 1);
      tc::mbar_init(&ctl->tmem_empty[b], PAIR ? 2 * EPI_WARPS : EPI_WARPS);
    }
    tc::mbar_init(&ctl->drain, 1);
    ctl->abort = 0;
    tc::fence_barrier_init();
  }
  if (warp == EPI_WARPS && lane == 0) {
    tc::tma_prefetch_desc(&tm_a);
    tc::tma_prefetch_desc(&tm_b);
  }
  if (warp == 0) {
    if constexpr (PAIR)
      tc::tmem_alloc_pair(&ctl->tmem, S::kTmem);
    else
      tc::tmem_alloc(&ctl->tmem, S::kTmem);
  }
  tc::tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) tc::cluster_sync();
  tc::tc_fence_after();
  const uint32_t tmem = ctl->tmem;
  pdl_wait();

  if (warp == EPI_WARPS) {
    // ---- TMA producer -----------------------------------------------------
    if (lane == 0) {
      int64_t i = 0;
      bool ok = true;
      Walk walk = walk0;
      int64_t t;
      int kb0, kb1;
      const uint32_t full0 = PAIR ? tc::map_to_rank(&ctl->full[0], 0) : 0u;
      while (ok && walk.next(t, kb0, kb1)) {
        const int mt = (int)(t / j.n_tiles), nt = (int)(t % j.n_tiles);
        const int a0 = mt * S::kRows + (int)rank * BM;
        // B rows of this CTA: with SiLU in columns, gate rows and the up rows `channels` further
        // (PAIR: the leader the gate's, its partner the up's)
        const int b0 = SILU && TOK_ROWS ? nt * S::kOutCols + (int)rank * j.channels
                                        : nt * BN + (int)rank * (BN / 2);
        for (int kb = kb0; kb < kb1; ++kb, ++i) {
          const int s = (int)(i % NST);
          const uint32_t use = (uint32_t)(i / NST);
          if (use > 0 &&
              !tc::mbar_wait(&ctl->empty[s], (use - 1) & 1u, kWaitLimitNs, &ctl->abort)) {
            ok = false;
            break;
          }
          uint8_t* a = tiles + s * SB;
          uint8_t* b = a + S::kA;
          if constexpr (PAIR) {
            const uint32_t bar = full0 + (uint32_t)(s * sizeof(uint64_t));
            if (rank == 0) tc::mbar_arrive_expect_tx(&ctl->full[s], 2 * SB);
            tc::tma_load_2d_pair(a, &tm_a, kb * BK, a0, bar);
            tc::tma_load_2d_pair(b, &tm_b, kb * BK, b0, bar);
          } else {
            tc::mbar_arrive_expect_tx(&ctl->full[s], SB);
            tc::tma_load_2d(a, &tm_a, kb * BK, a0, &ctl->full[s]);
            if constexpr (S::NACC == 2)
              tc::tma_load_2d(a + BM * BK, &tm_a, kb * BK, j.channels + a0, &ctl->full[s]);
            tc::tma_load_2d(b, &tm_b, kb * BK, b0, &ctl->full[s]);
            if constexpr (SILU && TOK_ROWS)
              tc::tma_load_2d(b + S::kB / 2, &tm_b, kb * BK, j.channels + b0, &ctl->full[s]);
          }
        }
      }
      if (!ok) raise_fault(ctl, fault);
      // every copy has landed before the shared memory is given up
      if (!PAIR || rank == 0)
        for (int64_t q = i > NST ? i - NST : 0; q < i; ++q)
          tc::mbar_wait(&ctl->full[q % NST], (uint32_t)(q / NST) & 1u, kWaitLimitNs, nullptr);
    }
  } else if (warp == EPI_WARPS + 1) {
    // ---- MMA issuer ---------------------------------------------------------
    if (lane == 0 && rank == 0) {
      constexpr uint32_t idesc = idesc_i8(S::kRows, BN);
      int64_t i = 0;
      int n = 0;
      bool ok = true;
      Walk walk = walk0;
      int64_t t;
      int kb0, kb1;
      for (; ok && walk.next(t, kb0, kb1); ++n) {
        const int b = n & 1;
        const uint32_t use_b = (uint32_t)(n >> 1);
        if (use_b > 0 &&
            !tc::mbar_wait(&ctl->tmem_empty[b], (use_b - 1) & 1u, kWaitLimitNs, &ctl->abort)) {
          ok = false;
          break;
        }
        tc::tc_fence_after();
        const uint32_t d = tmem + (uint32_t)(b * S::kCols);
        for (int kb = kb0; kb < kb1; ++kb, ++i) {
          const int s = (int)(i % NST);
          if (!tc::mbar_wait(&ctl->full[s], (uint32_t)(i / NST) & 1u, kWaitLimitNs, &ctl->abort)) {
            ok = false;
            break;
          }
          tc::tc_fence_after();
          const uint32_t a_addr = tc::smem_u32(tiles + s * SB);
          const uint64_t ad = tc::umma_desc_sw128(a_addr);
          const uint64_t bd = tc::umma_desc_sw128(a_addr + S::kA);
#pragma unroll
          for (int k = 0; k < BK / 32; ++k) {
            const uint32_t acc = kb > kb0 || k > 0 ? 1u : 0u;
            umma_i8<PAIR>(d, ad + 2 * k, bd + 2 * k, idesc, acc);
            if constexpr (S::NACC == 2)
              umma_i8<PAIR>(d + BN, ad + 2 * k + (BM * BK >> 4), bd + 2 * k, idesc, acc);
          }
          if constexpr (PAIR)
            tc::umma_commit_pair_both(&ctl->empty[s]);
          else
            tc::umma_commit(&ctl->empty[s]);
        }
        if (ok) {
          if constexpr (PAIR)
            tc::umma_commit_pair_both(&ctl->tmem_full[b]);
          else
            tc::umma_commit(&ctl->tmem_full[b]);
        }
      }
      if (!ok) raise_fault(ctl, fault);
      // every MMA has completed before TMEM is freed
      if constexpr (PAIR)
        tc::umma_commit_pair(&ctl->drain);
      else
        tc::umma_commit(&ctl->drain);
      tc::mbar_wait(&ctl->drain, 0, kWaitLimitNs, nullptr);
    }
  } else {
    // ---- epilogue: warp w drains lanes 32 (w % 4) .. +31, half w / 4 of the columns --------
    const int row = (warp % 4) * 32 + lane, c_begin = (warp / 4) * S::kHalf;
    const uint32_t tmem_empty0 = PAIR ? tc::map_to_rank(&ctl->tmem_empty[0], 0) : 0u;
    int n = 0;
    Walk walk = walk0;
    int64_t t;
    int kb0, kb1;
    for (; walk.next(t, kb0, kb1); ++n) {
      const int b = n & 1;
      const int mt = (int)(t / j.n_tiles), nt = (int)(t % j.n_tiles);
      const int m = mt * S::kRows + (int)rank * BM + row;  // this thread's token or channel
      const int c0 = nt * S::kOutCols;                     // the tile's first column
      const int rows_all = TOK_ROWS ? j.tokens : j.channels;
      const int cols_all = TOK_ROWS ? j.channels : j.tokens;
      const bool valid = m < rows_all;
      const bool whole = kb0 == 0 && kb1 == j.k_blocks;
      float s_row = 0.f, s_row2 = 0.f;
      float bias_row = 0.f;
      if (valid) {
        s_row = TOK_ROWS ? j.token_scales[m] : j.channel_scales[m];
        if (S::NACC == 2) s_row2 = j.channel_scales[j.channels + m];
        if (!TOK_ROWS && j.bias) bias_row = Traits<T>::to_f(static_cast<const T*>(j.bias)[m]);
      }
      bool ready = tc::mbar_wait(&ctl->tmem_full[b], (uint32_t)(n >> 1) & 1u, kWaitLimitNs,
                                 &ctl->abort);
      ready = epi_all(ready);
      if (!ready) {
        raise_fault(ctl, fault);
        break;
      }
      tc::tc_fence_after();
      const uint32_t acc = tmem + (uint32_t)(b * S::kCols) + ((uint32_t)(warp % 4 * 32) << 16);
      // the second accumulator (SiLU): the up columns
      constexpr int kUp = SILU ? (TOK_ROWS ? BN / 2 : BN) : 0;
      int w0 = 0, w1 = 0;  // the tile's workers
      bool finish = true;
      if (!whole) {
        const int64_t u0 = (t - t_stop) * j.k_blocks;
        w0 = sp.owner(u0);
        w1 = sp.owner(u0 + j.k_blocks - 1);
        // slot 0: the part that begins the tile, 1: one that goes on with it
        int32_t* slot = slots + ((int64_t)cta * 2 + (kb0 == 0 ? 0 : 1)) * S::kSlot;
#pragma unroll 1
        for (int c = c_begin; c < c_begin + S::kHalf && c0 + c < cols_all; c += CH) {
          __syncwarp();
#pragma unroll
          for (int up = 0; up <= kUp; up += kUp ? kUp : 1) {
            uint32_t r[CH];
            tmem_load(acc + (uint32_t)(c + up), r);
            tc::tmem_wait_ld(r);
            if (valid) store_partial(slot, c + up, row, r);
          }
        }
        // the last of the tile's workers finishes it.  A pair's CTAs have rows of their own
        epi_sync();
        if (threadIdx.x == 0) {
          int32_t* counter = counters + (t - t_stop) * (PAIR ? 2 : 1) + rank;
          uint32_t before;
          asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;"
                       : "=r"(before)
                       : "l"(counter)
                       : "memory");
          const bool last = before == (uint32_t)(w1 - w0);
          if (last) *counter = 0;
          ctl->last = last;
        }
        epi_sync();
        finish = *reinterpret_cast<volatile int*>(&ctl->last) != 0;
      }
      if (finish) {
#pragma unroll 1
        for (int c = c_begin; c < c_begin + S::kHalf && c0 + c < cols_all; c += CH) {
          __syncwarp();
          uint32_t r[CH], r2[CH];
          tmem_load(acc + (uint32_t)c, r);
          if (SILU) tmem_load(acc + (uint32_t)(c + kUp), r2);
          tc::tmem_wait_ld(r);
          if (SILU) tc::tmem_wait_ld(r2);
          if (!valid) continue;
          if (!whole) {
            for (int w = w0; w <= w1; ++w) {
              if (w == worker) continue;
              const int32_t* slot =
                  slots + ((int64_t)(PAIR ? 2 * w + (int)rank : w) * 2 + (w == w0 ? 0 : 1)) * S::kSlot;
              add_partial(slot, c, row, r);
              if (SILU) add_partial(slot, c + kUp, row, r2);
            }
          }
          if constexpr (TOK_ROWS) {
            const int ch = c0 + c;
            float y[CH];
#pragma unroll
            for (int e = 0; e < CH; ++e) {
              const int col = min(ch + e, j.channels - 1);
              y[e] = (float)(int)r[e] * s_row * __ldg(j.channel_scales + col);
              if (!SILU && j.bias) y[e] += Traits<T>::to_f(static_cast<const T*>(j.bias)[col]);
              if (SILU)
                y[e] = silu_mul<T>(
                    y[e], (float)(int)r2[e] * s_row * __ldg(j.channel_scales + j.channels + col));
            }
            put_channels<T, CH>(j, m, ch, y);
          } else {
#pragma unroll
            for (int e = 0; e < CH; ++e) {
              const int tok = c0 + c + e;
              if (tok >= j.tokens) break;
              const float st = __ldg(j.token_scales + tok);
              float y = (float)(int)r[e] * st * s_row + bias_row;
              if (SILU) y = silu_mul<T>(y, (float)(int)r2[e] * st * s_row2);
              if (j.add)
                y += Traits<T>::to_f(static_cast<const T*>(j.add)[tok * j.add_stride + m]);
              static_cast<T*>(j.out)[tok * j.out_stride + m] = Traits<T>::from_f(y);
            }
          }
        }
      }
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (PAIR)
          tc::mbar_arrive_cluster(tmem_empty0 + (uint32_t)(b * sizeof(uint64_t)));
        else
          tc::mbar_arrive(&ctl->tmem_empty[b]);
      }
    }
  }

  tc::tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) {
    tc::cluster_sync();
    if (warp == 0) tc::tmem_dealloc_pair(tmem, S::kTmem);
  } else {
    if (warp == 0) tc::tmem_dealloc(tmem, S::kTmem);
  }
}

// ------------------------------------------------------------ CUDA cores --
// Any K, stride and alignment: 32 tokens x 64 channels a CTA, 64 bytes of K at a
// time through shared memory, four products an instruction.
constexpr int kDotK = 64, kDotTok = 32, kDotCh = 64;

template <typename T, bool SILU>
__global__ void __launch_bounds__(256)
    int8_dot_kernel(const int8_t* __restrict__ codes, int64_t codes_stride,
                    const int8_t* __restrict__ weight, int64_t weight_stride, int k,
                    const GemmJob j) {
  constexpr int NW = SILU ? 2 : 1;
  __shared__ __align__(16) int8_t xs[kDotTok][kDotK + 4];
  __shared__ __align__(16) int8_t ws[NW][kDotCh][kDotK + 4];
  const int64_t t0 = (int64_t)blockIdx.y * kDotTok;
  const int n0 = (int)blockIdx.x * kDotCh;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;  // 4 channels, 2 tokens each
  pdl_launch_dependents();
  pdl_wait();
  int acc[NW][2][4] = {};
  for (int k0 = 0; k0 < k; k0 += kDotK) {
    for (int i = threadIdx.x; i < kDotTok * kDotK; i += 256) {
      const int r = i / kDotK, c = i % kDotK;
      xs[r][c] = t0 + r < j.tokens && k0 + c < k ? codes[(t0 + r) * codes_stride + k0 + c] : (int8_t)0;
    }
#pragma unroll
    for (int h = 0; h < NW; ++h)
      for (int i = threadIdx.x; i < kDotCh * kDotK; i += 256) {
        const int r = i / kDotK, c = i % kDotK;
        ws[h][r][c] = n0 + r < j.channels && k0 + c < k
                          ? weight[((int64_t)h * j.channels + n0 + r) * weight_stride + k0 + c]
                          : (int8_t)0;
      }
    __syncthreads();
#pragma unroll 4
    for (int c = 0; c < kDotK; c += 4) {
      int x[2];
#pragma unroll
      for (int a = 0; a < 2; ++a) x[a] = *reinterpret_cast<const int*>(&xs[ty * 2 + a][c]);
#pragma unroll
      for (int h = 0; h < NW; ++h)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const int w = *reinterpret_cast<const int*>(&ws[h][tx + 16 * b][c]);
#pragma unroll
          for (int a = 0; a < 2; ++a) acc[h][a][b] = __dp4a(x[a], w, acc[h][a][b]);
        }
    }
    __syncthreads();
  }
#pragma unroll
  for (int a = 0; a < 2; ++a) {
    const int64_t t = t0 + ty * 2 + a;
    if (t >= j.tokens) continue;
    const float st = j.token_scales[t];
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const int n = n0 + tx + 16 * b;
      if (n >= j.channels) continue;
      float y = (float)acc[0][a][b] * st * j.channel_scales[n];
      if (SILU)
        y = silu_mul<T>(y, (float)acc[NW - 1][a][b] * st * j.channel_scales[j.channels + n]);
      else if (j.bias)
        y += Traits<T>::to_f(static_cast<const T*>(j.bias)[n]);
      if (j.add) y += Traits<T>::to_f(static_cast<const T*>(j.add)[t * j.add_stride + n]);
      static_cast<T*>(j.out)[t * j.out_stride + n] = Traits<T>::from_f(y);
    }
  }
}

// -------------------------------------------------------------- host side --
struct Call {
  const int8_t *codes, *weight;
  int64_t codes_stride, weight_stride, tokens, k, channels;
  bool silu;
  void* workspace;
  size_t workspace_bytes;
  int32_t* fault;
  int dtype, device;
  cudaStream_t stream;
  const char* name;
};

// How the tokens lie in the tiles.  Up to 64 they are columns (16, 32 or 64 of
// them); above that rows, of a CTA pair where more than 128.
enum Way { kCols16, kCols32, kCols64, kRows128, kRows256 };
inline Way way_of(int64_t tokens) {
  if (tokens <= 16) return kCols16;
  if (tokens <= 32) return kCols32;
  if (tokens <= 64) return kCols64;
  return tokens <= 128 ? kRows128 : kRows256;
}

// A worker's least share of a tile that is cut, in K blocks.
constexpr int kLeastBlocks = 4;

struct Plan {
  int m_tiles, n_tiles, k_blocks, workers, split_workers;
  size_t slot_bytes;  // of all workers' partial sums
};

template <class S>
inline Plan plan_of(int64_t tokens, int64_t channels, int64_t k, int sms) {
  Plan p;
  const int64_t rows = S::TOK_ROWS ? tokens : channels, cols = S::TOK_ROWS ? channels : tokens;
  p.m_tiles = (int)ceil_div(rows, S::kRows);
  p.n_tiles = (int)ceil_div(cols, S::kOutCols);
  p.k_blocks = (int)ceil_div(k, BK);
  const int64_t all = (int64_t)p.m_tiles * p.n_tiles;
  const int most = std::max(1, S::PAIR ? sms / 2 : sms);
  // all workers take whole tiles; those left over are cut over as many workers as have
  // kLeastBlocks each
  const int64_t left = all % most;
  const int64_t units = left * p.k_blocks;
  int64_t cut = std::min<int64_t>(most, std::max(left, units / kLeastBlocks));
  if (cut == left && left > 0) cut = left;
  p.split_workers = (int)cut;
  p.workers = all < most ? (int)std::max<int64_t>(1, cut) : most;
  // whole tiles are dealt to `workers`, so with fewer than `most` none is whole
  p.slot_bytes = left == 0 || cut == left
                     ? 0
                     : (size_t)p.split_workers * (S::PAIR ? 2 : 1) * 2 * S::kSlot * sizeof(int32_t);
  return p;
}

template <class S>
size_t workspace_of(int64_t tokens, int64_t channels, int64_t k, int sms) {
  const Plan p = plan_of<S>(tokens, channels, k, sms);
  return p.slot_bytes ? (size_t)kCounterBytes + p.slot_bytes : 0;
}

int make_map(CUtensorMap* map, const int8_t* base, int64_t rows, int64_t k, int64_t stride, int box,
             const char* name) {
  tc::EncodeTiledFn enc = tc::encode_tiled();
  if (!enc) return fail(PACE_ERR_CUDA, "%s: cuTensorMapEncodeTiled unavailable", name);
  const cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)stride};
  const cuuint32_t boxes[2] = {(cuuint32_t)BK, (cuuint32_t)box};
  const cuuint32_t steps[2] = {1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t*>(base), dims,
                         strides, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(PACE_ERR_INVALID_ARGUMENT, "%s: tensor map rejected (CUresult %d)", name, (int)r);
  return PACE_OK;
}

template <typename T, class S>
int launch_gemm(const Call& c, GemmJob j) {
  const Plan p = plan_of<S>(c.tokens, c.channels, c.k, sm_count(c.device));
  if (p.slot_bytes && (!c.workspace || c.workspace_bytes < kCounterBytes + p.slot_bytes ||
                       !aligned16(c.workspace)))
    return fail(PACE_ERR_INVALID_ARGUMENT, "%s: workspace of %zu bytes (16-byte aligned) needed",
                c.name, (size_t)kCounterBytes + p.slot_bytes);
  j.m_tiles = p.m_tiles;
  j.n_tiles = p.n_tiles;
  j.k_blocks = p.k_blocks;
  const int64_t w_rows = c.silu ? 2 * c.channels : c.channels;
  CUtensorMap tok, ch;
  constexpr int kTokBox = S::TOK_ROWS ? BM : S::BN;
  constexpr int kChBox = S::TOK_ROWS ? (S::PAIR || S::SILU ? S::BN / 2 : S::BN) : BM;
  int rc = make_map(&tok, c.codes, c.tokens, c.k, c.codes_stride, kTokBox, c.name);
  if (rc == PACE_OK) rc = make_map(&ch, c.weight, w_rows, c.k, c.weight_stride, kChBox, c.name);
  if (rc != PACE_OK) return rc;
  auto kernel = int8_gemm_kernel<T, S>;
  cudaError_t err = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), c.device, S::kSmem);
  if (err != cudaSuccess) return cuda_fail(err, c.name);
  int32_t* counters = static_cast<int32_t*>(c.workspace);
  int32_t* slots = counters ? counters + kCounterBytes / 4 : nullptr;
  const CUtensorMap& a = S::TOK_ROWS ? tok : ch;
  const CUtensorMap& b = S::TOK_ROWS ? ch : tok;
  if constexpr (S::PAIR)
    err = launch_pairs(kernel, dim3((unsigned)(2 * p.workers)), dim3(THREADS), S::kSmem, c.stream,
                       a, b, j, p.split_workers, counters, slots, c.fault);
  else
    err = launch(kernel, dim3((unsigned)p.workers), dim3(THREADS), S::kSmem, c.stream, a, b, j,
                 p.split_workers, counters, slots, c.fault);
  return err == cudaSuccess ? PACE_OK : cuda_fail(err, c.name);
}

// Calls f.template operator()<Shape>() for the tokens' way.
template <bool SILU, typename F>
auto with_shape(int64_t tokens, F f) {
  switch (way_of(tokens)) {
    case kCols16: return f(Shape<16, false, false, SILU>{});
    case kCols32: return f(Shape<32, false, false, SILU>{});
    case kCols64: return f(Shape<64, false, false, SILU>{});
    case kRows128: return f(Shape<256, false, true, SILU>{});
    default: return f(Shape<256, true, true, SILU>{});
  }
}

// Whether TMA takes both operands.
inline bool for_tma(const Call& c) {
  return c.k % 16 == 0 && c.codes_stride % 16 == 0 && c.weight_stride % 16 == 0 &&
         aligned16(c.codes) && aligned16(c.weight);
}

template <typename T>
int run_typed(const Call& c, GemmJob j) {
  constexpr int V = Traits<T>::kVec;
  j.vec = aligned16(j.out) && j.out_stride % V == 0 &&
          (!j.add || (aligned16(j.add) && j.add_stride % V == 0));
  if (for_tma(c)) {
    auto go = [&](auto s) { return launch_gemm<T, decltype(s)>(c, j); };
    return c.silu ? with_shape<true>(c.tokens, go) : with_shape<false>(c.tokens, go);
  }
  const dim3 grid((unsigned)ceil_div(c.channels, kDotCh), (unsigned)ceil_div(c.tokens, kDotTok));
  if (ceil_div(c.tokens, kDotTok) > 65535)
    return fail(PACE_ERR_TOO_LARGE, "%s: over 2097120 tokens of rows that are not 16-byte aligned",
                c.name);
  const cudaError_t err =
      c.silu ? launch(int8_dot_kernel<T, true>, grid, dim3(256), 0, c.stream, c.codes,
                      c.codes_stride, c.weight, c.weight_stride, (int)c.k, j)
             : launch(int8_dot_kernel<T, false>, grid, dim3(256), 0, c.stream, c.codes,
                      c.codes_stride, c.weight, c.weight_stride, (int)c.k, j);
  return err == cudaSuccess ? PACE_OK : cuda_fail(err, c.name);
}

int run_int8(Call c, GemmJob j) {
  if (c.tokens < 0 || c.tokens > INT32_MAX || c.channels <= 0 || c.channels > (1 << 30) || c.k <= 0)
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
  j.tokens = (int)c.tokens;
  j.channels = (int)c.channels;
  return PACE_DISPATCH_FLOAT(c.dtype, c.name, [&] { return run_typed<scalar_t>(c, j); });
}

}  // namespace
}  // namespace pace

extern "C" size_t pace_int8_linear_workspace_size(int64_t num_tokens, int64_t out_features,
                                                  int64_t k, int gated, int device) {
  using namespace pace;
  if (num_tokens <= 0 || num_tokens > INT32_MAX || out_features <= 0 ||
      out_features > (1 << 30) || k <= 0 || k > kMaxK)
    return 0;
  const int sms = sm_count(device);
  auto go = [&](auto s) { return workspace_of<decltype(s)>(num_tokens, out_features, k, sms); };
  return gated ? with_shape<true>(num_tokens, go) : with_shape<false>(num_tokens, go);
}

extern "C" int pace_int8_linear(void* out, const int8_t* codes, const float* token_scales,
                                const int8_t* weight, const float* channel_scales,
                                const void* bias, const void* residual, int64_t num_tokens,
                                int64_t out_features, int64_t k, int64_t codes_row_stride,
                                int64_t weight_row_stride, int64_t out_row_stride,
                                int64_t residual_row_stride, int dtype, void* workspace,
                                size_t workspace_bytes, int32_t* fault_flags,
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
                         out_features, false, workspace, workspace_bytes, fault_flags, dtype, 0,
                         stream, "int8_linear"},
                        j);
}

extern "C" int pace_int8_gate_up_silu(void* out, const int8_t* codes, const float* token_scales,
                                      const int8_t* weight, const float* channel_scales,
                                      int64_t num_tokens, int64_t intermediate_size, int64_t k,
                                      int64_t codes_row_stride, int64_t weight_row_stride,
                                      int64_t out_row_stride, int dtype, void* workspace,
                                      size_t workspace_bytes, int32_t* fault_flags,
                                      cudaStream_t stream) {
  pace::GemmJob j = {};
  j.out = out;
  j.token_scales = token_scales;
  j.channel_scales = channel_scales;
  j.out_stride = out_row_stride;
  return pace::run_int8({codes, weight, codes_row_stride, weight_row_stride, num_tokens, k,
                         intermediate_size, true, workspace, workspace_bytes, fault_flags, dtype, 0,
                         stream, "int8_gate_up_silu"},
                        j);
}
