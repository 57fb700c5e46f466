// Paged attention of many query rows on the tensor cores (tcgen05): prompts,
// prompt chunks, draft trees and wide groups of heads.
//
// A CTA takes one piece of the plan for one kv head: up to 256 query rows
// (tokens x the group's heads, so that grouped heads share every key they
// read) in two tiles of 128, over keys [kv_begin, kv_end) in steps of 128.
//   S_t = Q_t K^T      128 x 128 per tile and step, accumulated in TMEM;
//   softmax            one thread per row: the row's 128 scores come from TMEM
//                      into registers, P goes back over them as 16-bit values;
//   O_t += P_t V       A operand from TMEM, O_t stays in TMEM throughout.
// Warps 0-3 and 4-7 are the two tiles' softmax, warp 8 issues the MMAs, the
// others copy K and V from their pages into a ring of 128-key tiles.  While one
// tile's rows are in softmax the tensor core works on the other tile.
//
// The running maximum m is allowed to lag: O and the sum l are scaled down only
// when a row's maximum has risen by more than 2^8 (kLag), so P is at most 2^8,
// which both 16-bit types hold with the same relative error, and O is read
// back and rescaled in a step of a sequence or two instead of in every one.
// S_t of step j + 1 is issued behind P_t V of step j, so its arrival also says
// that O_t may be touched.
//
// Keys outside the piece are copied as zeros, or as whatever codes lie there with
// a factor that makes them finite.  Every wait is bounded.
//
// What bounds it is the chain of a tile's step (scores out of TMEM, maximum,
// exponentials, P into TMEM, its product, the next scores): 3870 cycles for a step
// of both tiles, whose MMAs take about 2300.  One 8192-token prompt of 32 / 8 heads
// of 128, causal: 493 us in short runs, 1.12 PFLOP/s, 0.66 of cuBLAS's measured burst
// rate (570 us in long runs, under the power cap); with capped scores or distance
// bias 610 to 645 us (672), over a quantised cache 690 (703).
#include "attention_mma.cuh"
#include "tcgen05.cuh"

namespace pace {
namespace attn {

constexpr uint64_t kWaitLimitNs = 1000000000ull;  // 1 s per wait
constexpr int32_t kFaultTimeout = 1 << 30;
constexpr int kTileRowsEach = 128;
constexpr int kStepKeys = 128;
constexpr float kLag = 8.f;  // in powers of two
constexpr int kLoadBarrier = 1;

template <int D, bool Q8>
struct TileCfg {
  static constexpr int kLoadWarp0 = Q8 ? 12 : 9;
  static constexpr int kLoaders = Q8 ? 128 : 96;  // threads
  static constexpr int kThreads = kLoadWarp0 * 32 + kLoaders;
  static constexpr int kKvBytes = kStepKeys * D * 2;
  static constexpr int kQBytes = kTileRowsEach * D * 2;
  static constexpr int kStages = D == 64 ? 8 : Q8 ? 4 : 5;
  // a quantised cache's codes, as copied: K or V of a step
  static constexpr int kCodeBytes = kStepKeys * D;
  static constexpr int kCodeStages = 2;  // of TileCtl
  static constexpr int kCodeRingBytes = Q8 ? kCodeStages * kCodeBytes : 0;
  static constexpr int kSmemBytes =
      2 * kQBytes + kStages * kKvBytes + kCodeRingBytes + 1024 + 2048;
  // registers per thread after the split; the sum over the warpgroups is what
  // the block was launched with
  static constexpr int kSoftmaxRegs = Q8 ? 176 : 208;
  static constexpr int kOtherRegs = Q8 ? 80 : 88;
};

struct TileCtl {
  uint64_t q_full[2], s_full[2], p_full[2][2], o_full[2];
  uint64_t kv_full[8], kv_empty[8];
  uint64_t code_full[2], code_empty[2];
  uint64_t drain;
  uint32_t tmem;
  int abort;
  bool last;
  uint8_t exps[2][kStepKeys];   // exponents of the keys of a slot of codes
  uint32_t rows[kStepKeys];     // cache row (K part) of each key of a step; ~0: none
};
static_assert(sizeof(TileCtl) <= 2048, "");

__device__ __forceinline__ void tile_fault(TileCtl* ctl, int32_t* fault) {
  *reinterpret_cast<volatile int*>(&ctl->abort) = 1;
  if (fault) atomicOr(fault, kFaultTimeout);
}

// tc::mbar_wait with the timer out of the way: its read takes longer than most of
// these waits, so it is looked at once in many tries.
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, const TileCtl* ctl) {
  if (tc::mbar_try_wait(bar, parity)) return true;
  uint64_t t0 = 0;
  while (true) {
#pragma unroll 1
    for (int i = 0; i < 128; ++i)
      if (tc::mbar_try_wait(bar, parity)) return true;
    if (*reinterpret_cast<const volatile int*>(&ctl->abort)) return false;
    const uint64_t t = tc::globaltimer_ns();
    if (t0 == 0) t0 = t;
    if (t - t0 > kWaitLimitNs) return false;
  }
}

// Byte offset of 16-byte chunk `c` (8 dimensions) of row r of a 128-row tile:
// 64 dimensions a half, 128-byte rows, the chunk swizzled by the row.
__device__ __forceinline__ int tile_at(int r, int c) {
  return (c >> 3) * (128 * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}

// Operand descriptors are passed as their low words (start address and leading
// offset); the high words are constants: stride 1024 bytes (8 rows of 128),
// version 1, 128-byte swizzle.  K-major tiles (Q, K) ignore the leading offset.
// A V tile is MN-major: its rows are keys (the K axis of P V) of 64 contiguous
// dimensions, groups of 8 keys 1024 bytes apart, the next 64 dimensions 16 KB
// apart (the leading offset).
constexpr uint32_t kDescHigh = (1024u >> 4) | 1u << 14 | 2u << 29;
constexpr uint32_t kDescLeadK = 1u << 16, kDescLeadV = (16384u >> 4) << 16;

// D[tmem] (+)= A[smem] * B[smem]^T
__device__ __forceinline__ void umma_ss(uint32_t tmem_d, uint32_t a_low, uint32_t b_low,
                                        uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
      "mov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(a_low), "r"(b_low), "r"(idesc), "r"(accumulate), "n"(kDescHigh)
      : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem], B MN-major by its instruction descriptor.
__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint32_t b_low,
                                        uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
      "mov.b64 b, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "r"(b_low), "r"(idesc), "r"(accumulate), "n"(kDescHigh)
      : "memory");
}
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r)::"memory");
  return r != 0;
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
      "%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// Pairs of fp32 in one instruction.
__device__ __forceinline__ uint64_t u32x2(uint32_t lo, uint32_t hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
  return r;
}
__device__ __forceinline__ uint64_t f32x2(float lo, float hi) {
  return u32x2(__float_as_uint(lo), __float_as_uint(hi));
}
__device__ __forceinline__ float lo_of(uint64_t x) { return __uint_as_float((uint32_t)x); }
__device__ __forceinline__ float hi_of(uint64_t x) { return __uint_as_float((uint32_t)(x >> 32)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// The largest of three.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t both(float x) { return f32x2(x, x); }

// tanh(u) / u on |u| <= 1 as a polynomial in z = u^2, fitted for the least
// largest error of tanh (2.5e-7: in the score, 1.3e-5 of a cap of 50).
__device__ __forceinline__ uint64_t tanh_ratio_pair(uint64_t z) {
  uint64_t y = fma2(both(-0.002840145258232951f), z, both(0.016116151586174965f));
  y = fma2(y, z, both(-0.05097497999668121f));
  y = fma2(y, z, both(0.13253627717494965f));
  y = fma2(y, z, both(-0.33324024081230164f));
  return fma2(y, z, both(0.9999968409538269f));
}
__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
// One box of a page: `slots` keys of one head, 64 dimensions, swizzled.
__device__ __forceinline__ void tma_load_page(void* dst, const CUtensorMap* map, int dim, int head,
                                              int slot, int page_kind, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(tc::smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(dim), "r"(head), "r"(slot), "r"(page_kind),
      "r"(tc::smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void fence_async_proxy() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

__device__ __forceinline__ void mbar_arrive_many(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(tc::smem_u32(bar)), "r"(count)
               : "memory");
}

// Barrier of the copying threads that also ANDs `pred` over them.
template <int N>
__device__ __forceinline__ bool loaders_all(bool pred) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "bar.red.and.pred q, %2, %3, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(pred ? 1u : 0u), "n"(kLoadBarrier), "n"(N)
      : "memory");
  return r != 0;
}

// Bits of the keys j0 .. j0 + 31 that a row sees: lo <= j < hi, and of the
// drafted ones base .. end - 1 those of its tree row.
__device__ __forceinline__ uint32_t seen_bits(int j0, int lo, int hi, int base, int end,
                                              const uint64_t* tree) {
  auto below = [](int n) -> uint32_t {  // the first n bits
    return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u;
  };
  uint32_t bits = below(hi - j0) & ~below(lo - j0);
  if (tree && j0 + 32 > base && j0 < end) {
    const int n0 = j0 - base;  // node of bit 0
    uint32_t t;
    if (n0 < 0) {
      t = (uint32_t)tree[0] << -n0;  // -n0 < 32
    } else {
      const uint64_t w = tree[n0 >> 6];
      t = (uint32_t)(w >> (n0 & 63));
      // the next word, where the sequence reaches into it
      if ((n0 & 63) > 32 && base + ((n0 >> 6) + 1) * 64 < end)
        t |= (uint32_t)(tree[(n0 >> 6) + 1] << (64 - (n0 & 63)));
    }
    bits |= t & below(end - j0) & ~below(max(base, lo) - j0);
  }
  return bits;
}

template <typename T, int D, bool Q8>
__global__ void __launch_bounds__(TileCfg<D, Q8>::kThreads, 1)
    attention_tile_kernel(const Problem p, const __grid_constant__ CUtensorMap map, int box,
                          const Item* items, float* partial, float2* partial_ml,
                          int32_t* counters, int32_t* fault) {
  using Cfg = TileCfg<D, Q8>;
  using M = Mma<T>;
  constexpr float kUp = std::is_same<T, __half>::value ? kHeadroom : 0.f;  // of P and its sum
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* ring = smem + 2 * Cfg::kQBytes;
  uint8_t* codes = ring + Cfg::kStages * Cfg::kKvBytes;
  TileCtl* ctl = reinterpret_cast<TileCtl*>(codes + Cfg::kCodeRingBytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kvh = blockIdx.x % p.kv_heads;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&ctl->q_full[i], 128);
      tc::mbar_init(&ctl->s_full[i], 1);
      tc::mbar_init(&ctl->p_full[i][0], 4);
      tc::mbar_init(&ctl->p_full[i][1], 4);
      tc::mbar_init(&ctl->o_full[i], 1);
    }
    for (int i = 0; i < Cfg::kStages; ++i) {
      tc::mbar_init(&ctl->kv_full[i], Cfg::kLoaders);
      tc::mbar_init(&ctl->kv_empty[i], 1);
    }
    for (int i = 0; i < Cfg::kCodeStages; ++i) {
      tc::mbar_init(&ctl->code_full[i], 3);  // the codes' warp, two of the exponents
      tc::mbar_init(&ctl->code_empty[i], Cfg::kLoaders);
    }
    tc::mbar_init(&ctl->drain, 1);
    ctl->abort = 0;
    tc::fence_barrier_init();
  }
  if (warp == 8) tc::tmem_alloc(&ctl->tmem, 512);
  pdl_wait();
  // not earlier: a kernel may have written the plan.  Ahead of the barrier, which hides the latency
  // (8192 tokens 498 us, behind it 513), but for a quantised cache, whose roles have no registers
  // to spare for it (8192 tokens, capped: 846 us, behind it 832).
  Item w;
  if constexpr (!Q8) w = items[blockIdx.x / p.kv_heads];
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = ctl->tmem;
  // not before the wait: the few-row kernel of the same call starts beside this one without a wait
  // of its own, on what is complete here
  pdl_launch_dependents();
  if constexpr (Q8) w = items[blockIdx.x / p.kv_heads];
  const int group = p.heads / p.kv_heads;
  const int rows = w.ntok * group;
  // row / group for rows below 256 and groups up to 128: the fraction added stays below 1 / group
  const uint32_t group_inv = 65536u / (uint32_t)group + 1u;
  auto div_group = [&](int row) { return (int)((uint32_t)row * group_inv >> 16); };
  const int tiles = rows > kTileRowsEach ? 2 : 1;
  // steps lie on multiples of 128 keys, so that pages do not straddle them
  const int k_base = w.kv_begin & ~(kStepKeys - 1);
  const int steps = w.kv_end > w.kv_begin ? (w.kv_end - k_base + kStepKeys - 1) / kStepKeys : 0;

  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Cfg::kSoftmaxRegs));
    // ---- softmax of tile t: thread = row ---------------------------------------
    const int t = warp >> 2;
    const int r = threadIdx.x & 127;      // row of the tile
    const int row = t * kTileRowsEach + r;  // of the piece
    const bool live = row < rows;
    const int tok_of = live ? div_group(row) : 0;
    const int tok = w.tok0 + tok_of;
    const int head = kvh * group + (live ? row - tok_of * group : 0);
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    if (t < tiles) {
      // the tile's queries, a row by 8 or 16 neighbouring threads; negated where the scale is
      // negative (and zero where it is), so that the largest product is the largest score.  A piece
      // without a step leaves them: nothing would order these stores, all over the tile, before the
      // warps' outputs, which pass through the same memory.
      if (steps > 0) {
        uint8_t* qs = smem + t * Cfg::kQBytes;
        const uint32_t flip = p.scale < 0.f ? 0x80008000u : 0u;
        const bool vec = p.q_stride % 8 == 0 && (reinterpret_cast<uintptr_t>(p.query) & 15) == 0;
        constexpr int kChunks = D / 8, kRowStep = 128 / kChunks;
        const int c = r % kChunks;
        uint4 q[kChunks];  // all loads first, then the stores
#pragma unroll
        for (int x = 0; x < kChunks; ++x) {
          const int at = t * kTileRowsEach + x * kRowStep + r / kChunks;
          q[x] = make_uint4(0, 0, 0, 0);
          if (at < rows && p.scale != 0.f) {
            const int tk = div_group(at);
            const T* src = static_cast<const T*>(p.query) + (int64_t)(w.tok0 + tk) * p.q_stride +
                           (int64_t)(kvh * group + at - tk * group) * D + c * 8;
            q[x] = vec ? ld_nc_v4(src)
                       : make_uint4(M::pair(src[0], src[1]), M::pair(src[2], src[3]),
                                    M::pair(src[4], src[5]), M::pair(src[6], src[7]));
          }
        }
#pragma unroll
        for (int x = 0; x < kChunks; ++x) {
          uint32_t v[4] = {q[x].x, q[x].y, q[x].z, q[x].w};
          if constexpr (Q8) {
            // quantised keys are unpacked as dimensions 0, 2, 1, 3 of each four
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
              const uint32_t a = v[i], b = v[i + 1];
              v[i] = __byte_perm(a, b, 0x5410);
              v[i + 1] = __byte_perm(a, b, 0x7632);
            }
          }
          *reinterpret_cast<uint4*>(qs + tile_at(x * kRowStep + r / kChunks, c)) =
              make_uint4(v[0] ^ flip, v[1] ^ flip, v[2] ^ flip, v[3] ^ flip);
        }
        fence_async_proxy();
        tc::mbar_arrive(&ctl->q_full[t]);
      }
      TokenInfo info{0, 0, 0, 0};
      float slope = 0.f;
      const uint64_t* tree = nullptr;
      if (live) {
        info = p.tokens[tok];
        if (p.slopes) slope = p.slopes[head] * kLog2e;
        if (p.tree_mask) tree = p.tree_mask + (int64_t)tok * p.tree_words;
      }
      const int end = tree ? min(info.pos, w.kv_end) : 0;  // of the drafted keys
      // a row that is none sees everything, which saves its warp the masks; nothing is made of it
      const int lo = live ? max(info.lo, w.kv_begin) : 0;
      const int hi = live ? min(info.hi, w.kv_end) : INT32_MAX;
      const float scale2 = (p.scale != 0.f ? fabsf(p.scale) : 1.f) * kLog2e;
      const float cap2 = p.cap * kLog2e, cap_in = p.cap > 0.f ? 2.f * scale2 / p.cap : 0.f;
      const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
      const uint32_t ts = tmem + lanes + (uint32_t)(t * 128);
      const uint32_t to = tmem + lanes + 256u + (uint32_t)(t * D);
      for (int j = 0; j < steps; ++j) {
        ok = __all_sync(0xffffffffu,
                        wait_for(&ctl->s_full[t], j & 1, ctl));
        if (!ok) break;
        // the last tile's scores are the last reader of K of this step and come behind the last
        // reader of V of the step before: their slots are free.  Said here, not by commits of the
        // MMA warp, each of which would hold up its next MMA.
        if (t == tiles - 1 && r == 0) {
          tc::mbar_arrive(&ctl->kv_empty[(2 * j) % Cfg::kStages]);
          if (j > 0) tc::mbar_arrive(&ctl->kv_empty[(2 * j - 1) % Cfg::kStages]);
        }
        tc::tc_fence_after();
        uint32_t sr[128];
        tmem_ld32(ts, sr);
        tmem_ld32(ts + 32, sr + 32);
        tmem_ld32(ts + 64, sr + 64);
        tmem_ld32(ts + 96, sr + 96);
        tc::tmem_wait_ld(sr);
        float sc = scale2;
        const int j0 = k_base + j * kStepKeys;
        if (p.cap > 0.f) {
          float size[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 0; i < kStepKeys; i += 8)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              size[k] = max3(size[k], fabsf(__uint_as_float(sr[i + 2 * k])),
                             fabsf(__uint_as_float(sr[i + 2 * k + 1])));
          size[0] = fmaxf(fmaxf(size[0], size[1]), fmaxf(size[2], size[3]));
          if (__all_sync(0xffffffffu, size[0] * scale2 <= 0.25f * cap2)) {
            // all scores well within the cap, as they mostly are: three terms of the polynomial
            // (largest error of tanh 5.0e-8), the factors in its coefficients.  8192 tokens, capped:
            // 631 us, 740 with the six terms below, 1026 with the special-function unit.
            const float in = scale2 / cap2, z1 = in * in;
            const uint64_t a0 = both(0.9999986290931702f * scale2);
            const uint64_t a1 = both(-0.3331570625305176f * scale2 * z1);
            const uint64_t a2 = both(0.12762290239334106f * scale2 * z1 * z1);
#pragma unroll
            for (int i = 0; i < kStepKeys; i += 2) {
              const uint64_t x = u32x2(sr[i], sr[i + 1]), z = mul2(x, x);
              const uint64_t y = mul2(x, fma2(fma2(a2, z, a1), z, a0));
              sr[i] = (uint32_t)y;
              sr[i + 1] = (uint32_t)(y >> 32);
            }
          } else if (__all_sync(0xffffffffu, size[0] * scale2 <= cap2)) {
            // no score passes the cap: tanh by a polynomial.  The special-function unit, which
            // two calls a score keep busy for longer than the exponentials do, has none of it.
            const uint64_t in2 = both(scale2 / cap2), out2 = both(scale2);
#pragma unroll
            for (int i = 0; i < kStepKeys; i += 2) {
              const uint64_t x = u32x2(sr[i], sr[i + 1]), u = mul2(x, in2);
              const uint64_t y = mul2(mul2(x, out2), tanh_ratio_pair(mul2(u, u)));
              sr[i] = (uint32_t)y;
              sr[i + 1] = (uint32_t)(y >> 32);
            }
          } else {
#pragma unroll
            for (int i = 0; i < kStepKeys; ++i)
              sr[i] = __float_as_uint(
                  cap2 -
                  2.f * cap2 * rcp_approx(1.f + exp2_approx(__uint_as_float(sr[i]) * cap_in)));
          }
          sc = 1.f;
        }
        if (p.slopes) {
          const float d0 = (float)(info.pos - j0);
          if (__all_sync(0xffffffffu, d0 >= (float)(kStepKeys - 1))) {
            // all keys lie before the row's token: the bias rises by the slope from key to key
            const uint64_t sc2 = both(sc);
            uint64_t rise[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
              rise[k] = f32x2(slope * (2.f * k - d0), slope * (2.f * k + 1.f - d0));
            const uint64_t by = both(8.f * slope);
#pragma unroll
            for (int i = 0; i < kStepKeys; i += 8)
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const int x = i + 2 * k;
                const uint64_t y = fma2(u32x2(sr[x], sr[x + 1]), sc2, rise[k]);
                rise[k] = add2(rise[k], by);
                sr[x] = (uint32_t)y;
                sr[x + 1] = (uint32_t)(y >> 32);
              }
          } else {
#pragma unroll
            for (int i = 0; i < kStepKeys; ++i)
              sr[i] = __float_as_uint(__uint_as_float(sr[i]) * sc - slope * fabsf(d0 - (float)i));
          }
          sc = 1.f;
        }
        const bool whole = j0 >= lo && j0 + kStepKeys <= hi;
        if (!__all_sync(0xffffffffu, whole)) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t bits = seen_bits(j0 + 32 * k, lo, min(hi, w.kv_end), info.hi, end, tree);
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!(bits >> i & 1)) sr[32 * k + i] = 0xff800000u;
          }
          __syncwarp();
        }
        float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 128; i += 8)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            tops[k] = max3(tops[k], __uint_as_float(sr[i + 2 * k]),
                           __uint_as_float(sr[i + 2 * k + 1]));
        float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
        top *= sc;
        if (j == 0) {
          m = top;
        } else {
          const bool raise = top > m + kLag || (m == -INFINITY && top > m);
          if (__any_sync(0xffffffffu, raise)) {
            // O is complete up to the step before: S of this step was issued behind it
            const float f = raise ? exp2_approx(m - top) : 1.f;
            if (raise) m = top;
            l *= f;
#pragma unroll
            for (int c = 0; c < D; c += 32) {
              uint32_t o[32];
              tmem_ld32(to + c, o);
              tc::tmem_wait_ld(o);
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
              tmem_st16(to + c, o);
              tmem_st16(to + c + 16, o + 16);
            }
          }
        }
        const float b = m == -INFINITY ? 0.f : m - kUp;
        uint64_t sum[2] = {0, 0};  // two pairs of partial sums
        const uint64_t sc2 = f32x2(sc, sc), b2 = f32x2(-b, -b);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const uint64_t z = fma2(u32x2(sr[32 * k + 2 * i], sr[32 * k + 2 * i + 1]), sc2, b2);
            const float x = exp2_approx(lo_of(z)), y = exp2_approx(hi_of(z));
            sum[i & 1] = add2(sum[i & 1], f32x2(x, y));
            pk[i] = M::pack(x, y);
          }
          tmem_st16(ts + 16 * k, pk);
          if (k & 1) {
            // half of P is in place: its product may begin
            tmem_wait_st();
            tc::tc_fence_before();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&ctl->p_full[t][k >> 1]);
          }
        }
        sum[0] = add2(sum[0], sum[1]);
        l += lo_of(sum[0]) + hi_of(sum[0]);
      }
      // ---- the tile's output ----------------------------------------------------
      m -= kUp;
      if (ok && steps > 0)
        ok = __all_sync(0xffffffffu,
                        wait_for(&ctl->o_full[t], 0, ctl));
      if (!ok) tile_fault(ctl, fault);
      if (ok) {
        tc::tc_fence_after();
        const int64_t slot = ((int64_t)(w.slot + w.split) * p.kv_heads + kvh) * 256 + row;
        const float inv = l == 0.f ? 0.f : 1.f / l;
        // whole rows go out through the query tile's place, so that a warp writes rows and not
        // 16 bytes of each of 32 rows
        uint8_t* os = smem + t * Cfg::kQBytes;
        float size = 0.f;
#pragma unroll
        for (int c = 0; c < D; c += 32) {
          uint32_t o[32];
          if (steps > 0) {
            tmem_ld32(to + c, o);
            tc::tmem_wait_ld(o);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0;
          }
          float v[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const int s = Q8 ? (i & ~3) | ((i & 1) << 1) | ((i >> 1) & 1) : i;
            v[i] = __uint_as_float(o[s]);
          }
          if (w.splits > 1) {
            float* dst = partial + slot * D + c;
            if (live) {
#pragma unroll
              for (int i = 0; i < 32; i += 8)
                st_v8(dst + i,
                      make_uint4(__float_as_uint(v[i]), __float_as_uint(v[i + 1]),
                                 __float_as_uint(v[i + 2]), __float_as_uint(v[i + 3])),
                      make_uint4(__float_as_uint(v[i + 4]), __float_as_uint(v[i + 5]),
                                 __float_as_uint(v[i + 6]), __float_as_uint(v[i + 7])));
            }
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              v[i] = l == 0.f ? 0.f : v[i] * inv;
              size += fabsf(v[i]);
            }
#pragma unroll
            for (int i = 0; i < 32; i += 8)
              *reinterpret_cast<uint4*>(os + tile_at(r, (c + i) / 8)) = Traits<T>::pack(v + i);
          }
          __syncwarp();
        }
        if (w.splits == 1) {
          // a warp's 32 rows are its own
          constexpr int kChunks = D / 8, kRowStep = 32 / kChunks;
          const int c = lane % kChunks;
          const bool vec = p.out_stride % 8 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0;
#pragma unroll 4
          for (int x = 0; x < kChunks; ++x) {
            const int qr = (warp & 3) * 32 + x * kRowStep + lane / kChunks;
            const int at = t * kTileRowsEach + qr;
            if (at < rows) {
              const int tk = div_group(at);
              T* dst = static_cast<T*>(p.out) + (int64_t)(w.tok0 + tk) * p.out_stride +
                       (int64_t)(kvh * group + at - tk * group) * D + c * 8;
              const uint4 y = *reinterpret_cast<const uint4*>(os + tile_at(qr, c));
              if (vec) {
                st_v4(dst, y);
              } else {
                const T* e = reinterpret_cast<const T*>(&y);
#pragma unroll
                for (int i = 0; i < 8; ++i) dst[i] = e[i];
              }
            }
          }
        }
        if (live) {
          if (w.splits > 1)
            __stcg(partial_ml + slot, make_float2(m, l));
          else if (p.lse)
            p.lse[(int64_t)tok * p.heads + head] =
                l == 0.f ? -INFINITY : m * 0.6931471805599453f + logf(l);
        }
        if (w.mixed && w.splits == 1) {
          // not where the sum, which no hidden key enters, is infinite or NaN as well
          uint32_t bad = __ballot_sync(0xffffffffu, live && l < INFINITY && !(size < INFINITY));
          if (bad) __syncwarp();  // their stores come before the ones below
          for (; bad; bad &= bad - 1) {
            const int at = row - lane + __ffs(bad) - 1;
            attend_row_again<T, Q8, D>(p, w.tok0 + at / group, kvh * group + at % group,
                                       w.all_begin, w.all_end, false);
          }
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Cfg::kOtherRegs));
    if (warp == 8) {
      // ---- MMA issuer: the whole warp walks the steps, so that descriptors and
      // addresses stay in uniform registers; one lane issues ---------------------------
      if (steps > 0) {
        constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
        constexpr uint32_t idesc_s = tc::umma_idesc_f16(kBf16, 128, kStepKeys);
        constexpr uint32_t idesc_o = tc::umma_idesc_f16(kBf16, 128, D) | (1u << 16);  // B MN-major
        constexpr uint32_t kSlot = Cfg::kKvBytes >> 4;
        const uint32_t q0 = (tc::smem_u32(smem) >> 4) | kDescLeadK;
        const uint32_t r0 = tc::smem_u32(ring) >> 4;
        const uint32_t ubase = __shfl_sync(0xffffffffu, tmem, 0);
        bool ok = true;
        auto wait = [&](uint64_t* bar, uint32_t parity) {
          ok = ok && wait_for(bar, parity, ctl);
          ok = __all_sync(0xffffffffu, ok);
          tc::tc_fence_after();
          return ok;
        };
        // ring slots in order: K of step 0, V of step 0, K of step 1, ...
        int ks = 0, vs = 1 % Cfg::kStages;  // slots of the next K and V
        uint32_t kp = 0, vp = 0;            // their phases
        auto step_slot = [](int& s, uint32_t& phase) {
          s += 2;
          if (s >= Cfg::kStages) {
            s -= Cfg::kStages;
            phase ^= 1u;
          }
        };
        auto scores = [&](int t, int slot) {
          if (elect_one()) {
            const uint32_t q = q0 + (uint32_t)t * (Cfg::kQBytes >> 4);
            const uint32_t k = (r0 + (uint32_t)slot * kSlot) | kDescLeadK;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
              const uint32_t at = (uint32_t)((i >> 2) * 16384 + (i & 3) * 32) >> 4;
              umma_ss(ubase + t * 128, q + at, k + at, idesc_s, i > 0);
            }
            tc::umma_commit(&ctl->s_full[t]);
          }
          __syncwarp();
        };
        auto output = [&](int t, int slot, int half, bool add) {
          if (elect_one()) {
            const uint32_t v = (r0 + (uint32_t)slot * kSlot) | kDescLeadV;
#pragma unroll
            for (int x = 0; x < kStepKeys / 32; ++x) {
              const int i = half * (kStepKeys / 32) + x;
              umma_ts(ubase + 256 + t * D, ubase + t * 128 + i * 8, v + (i * 2048 >> 4), idesc_o,
                      x > 0 || add);
            }
          }
          __syncwarp();
        };
        for (int t = 0; t < tiles; ++t) {
          if (!wait(&ctl->q_full[t], 0)) break;
          if (t == 0 && !wait(&ctl->kv_full[0], 0)) break;
          scores(t, 0);
        }
        step_slot(ks, kp);
        for (int j = 0; ok && j < steps; ++j) {
          if (!wait(&ctl->kv_full[vs], vp)) break;
          for (int t = 0; t < tiles; ++t) {
            if (!wait(&ctl->p_full[t][0], j & 1)) break;
            output(t, vs, 0, j > 0);
            if (!wait(&ctl->p_full[t][1], j & 1)) break;
            output(t, vs, 1, true);
            if (j + 1 < steps) {
              if (t == 0 && !wait(&ctl->kv_full[ks], kp)) break;
              scores(t, ks);
            } else if (elect_one()) {
              tc::umma_commit(&ctl->o_full[t]);
            }
          }
          step_slot(ks, kp);
          step_slot(vs, vp);
        }
        if (!ok) tile_fault(ctl, fault);
        if (elect_one()) {
          tc::umma_commit(&ctl->drain);
          tc::mbar_wait(&ctl->drain, 0, kWaitLimitNs, nullptr);
        }
        __syncwarp();
      }
    } else if (Q8 && box > 0 && warp < Cfg::kLoadWarp0) {
      // ---- quantised pages by TMA: codes (warp 9) and exponents (warps 10, 11) ------
      // Keys outside the piece get the exponent 0: whatever codes lie there, they
      // come out finite.
      bool ok = true;
      if (warp == 9) {
        int page = 0;
        constexpr int kBoxes = kStepKeys / 8;  // at most
        static_assert(kBoxes <= 32, "");
        const int key = lane * box;
        auto look_up = [&](int j) {
          const int pos = k_base + j * kStepKeys + key;
          return key < kStepKeys && pos < w.kv_end ? p.kv_indices[w.page_base + page_number(p, pos)] : -1;
        };
        page = look_up(0);
        int sent = 0;
        for (int i = 0; ok && i < 2 * steps; ++i) {
          const int s = i % Cfg::kCodeStages;
          if (i >= Cfg::kCodeStages)
            ok = __all_sync(0xffffffffu, wait_for(&ctl->code_empty[s],
                                                  (uint32_t)(i / Cfg::kCodeStages - 1) & 1u, ctl));
          if (!ok) break;
          const uint32_t there = __ballot_sync(0xffffffffu, page >= 0);
          if (lane == 0)
            tc::mbar_arrive_expect_tx(&ctl->code_full[s], (uint32_t)(__popc(there) * box * D));
          __syncwarp();
          if (page >= 0) {
            const int pos = k_base + (i >> 1) * kStepKeys + key;
            tma_load_page(codes + s * Cfg::kCodeBytes + key * D, &map, 0, kvh, page_slot(p, pos),
                          page * 2 + (i & 1), &ctl->code_full[s]);
          }
          sent = i + 1;
          if (i & 1) page = look_up((i >> 1) + 1);
        }
        // whatever ended the steps, no copy outlives the CTA
        for (int i = max(sent - Cfg::kCodeStages, 0); i < sent; ++i)
          tc::mbar_wait(&ctl->code_full[i % Cfg::kCodeStages],
                        (uint32_t)(i / Cfg::kCodeStages) & 1u, kWaitLimitNs, nullptr);
      } else {
        const int u = threadIdx.x - 10 * 32;  // keys u and u + 64 of each step
        const int64_t v_rows = (int64_t)p.page_size * p.kv_heads;
        auto row_of = [&](int j, int key) -> int64_t {
          const int pos = k_base + j * kStepKeys + key;
          if (j >= steps || pos < w.kv_begin || pos >= w.kv_end) return -1;
          const int64_t page = p.kv_indices[w.page_base + page_number(p, pos)];
          return (page * 2 * p.page_size + page_slot(p, pos)) * p.kv_heads + kvh;
        };
        // rows two steps ahead, exponents one step ahead: their loads depend on each other
        int64_t rows[2] = {row_of(0, u), row_of(0, u + 64)};
        uint8_t ex[2][2];
        auto load = [&]() {
#pragma unroll
          for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int kind = 0; kind < 2; ++kind)
              ex[kind][k] = rows[k] >= 0 ? p.exponents[rows[k] + kind * v_rows] : 0;
        };
        load();
        rows[0] = row_of(1, u);
        rows[1] = row_of(1, u + 64);
        for (int i = 0; ok && i < 2 * steps; ++i) {
          const int s = i % Cfg::kCodeStages;
          if (i >= Cfg::kCodeStages)
            ok = __all_sync(0xffffffffu, wait_for(&ctl->code_empty[s],
                                                  (uint32_t)(i / Cfg::kCodeStages - 1) & 1u, ctl));
          if (!ok) break;
          ctl->exps[s][u] = ex[i & 1][0];
          ctl->exps[s][u + 64] = ex[i & 1][1];
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(&ctl->code_full[s]);
          if (i & 1) {
            load();
            rows[0] = row_of((i >> 1) + 2, u);
            rows[1] = row_of((i >> 1) + 2, u + 64);
          }
        }
      }
      if (!ok) tile_fault(ctl, fault);
    } else if (Q8 && box > 0) {
      // ---- codes to 16-bit values, slot by slot -------------------------------------
      // A thread has one key, whose factor it finds once; the chunk it begins with goes
      // by the key, so that neighbours meet in no bank.
      constexpr int kChunks = D / 16;
      static_assert(Cfg::kLoaders == kStepKeys || !Q8, "");
      const int key = threadIdx.x - Cfg::kLoadWarp0 * 32;
      bool ok = true;
      for (int i = 0; ok && i < 2 * steps; ++i) {
        const int s = i % Cfg::kCodeStages, d = i % Cfg::kStages;
        ok = wait_for(&ctl->code_full[s], (uint32_t)(i / Cfg::kCodeStages) & 1u, ctl);
        if (ok && i >= Cfg::kStages)
          ok = wait_for(&ctl->kv_empty[d], (uint32_t)(i / Cfg::kStages - 1) & 1u, ctl);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const uint8_t* src = codes + s * Cfg::kCodeBytes + key * D;
        uint8_t* dst = ring + d * Cfg::kKvBytes;
        const uint32_t ex = ctl->exps[s][key];
        uint4 v[kChunks];
#pragma unroll
        for (int x = 0; x < kChunks; ++x)
          v[x] = *reinterpret_cast<const uint4*>(src + ((x + key) % kChunks) * 16);
#pragma unroll
        for (int x = 0; x < kChunks; ++x) {
          const int c = (x + key) % kChunks;
          const uint32_t w4[4] = {v[x].x, v[x].y, v[x].z, v[x].w};
          uint32_t o[8];
          M::dequantise16(w4, ex, o);
          *reinterpret_cast<uint4*>(dst + tile_at(key, 2 * c)) = make_uint4(o[0], o[1], o[2], o[3]);
          *reinterpret_cast<uint4*>(dst + tile_at(key, 2 * c + 1)) =
              make_uint4(o[4], o[5], o[6], o[7]);
        }
        fence_async_proxy();
        tc::mbar_arrive(&ctl->code_empty[s]);
        tc::mbar_arrive(&ctl->kv_full[d]);
      }
      if (!ok) tile_fault(ctl, fault);
    } else if (warp >= Cfg::kLoadWarp0) {
      // ---- copies: slot 2j is K, slot 2j + 1 V of step j ----------------------------
      // Whole steps come box by box through TMA, issued by the first of these warps
      // alone, where the pages allow it (box > 0).  The others, ragged ones among
      // them, take all threads: 16-byte copies (zeros for keys outside the piece) of
      // a 16-bit cache, loads and unpacking of a quantised one.
      constexpr int N = Cfg::kLoaders;
      const int u = threadIdx.x - Cfg::kLoadWarp0 * 32;
      const uint8_t* cache = static_cast<const uint8_t*>(p.cache);
      const int64_t v_rows = (int64_t)p.page_size * p.kv_heads;
      auto by_tma = [&](int j) {
        const int j0 = k_base + j * kStepKeys;
        return !Q8 && box > 0 && j0 >= w.kv_begin && j0 + kStepKeys <= w.kv_end;
      };
      constexpr int kHalves = D / 64;
      const int box_key = u / kHalves * (box > 0 ? box : 1), box_half = u % kHalves;
      const bool has_box = u < 32 && box > 0 && box_key < kStepKeys;
      auto page_of = [&](int j) {  // of this lane's box
        const int pos = k_base + j * kStepKeys + box_key;
        return has_box && j < steps && pos < w.kv_end ? p.kv_indices[w.page_base + page_number(p, pos)]
                                                      : 0;
      };
      int page = u < 32 ? page_of(0) : 0;
      auto row_of = [&](int j, int key) -> uint32_t {
        const int pos = k_base + j * kStepKeys + key;
        if (j >= steps || pos < w.kv_begin || pos >= w.kv_end) return ~0u;
        const int64_t page = p.kv_indices[w.page_base + page_number(p, pos)];
        return (uint32_t)((page * 2 * p.page_size + page_slot(p, pos)) * p.kv_heads + kvh);
      };
      constexpr int kOwn = (kStepKeys + N - 1) / N;  // keys whose row a thread looks up
      uint32_t next[kOwn];
      auto look_up = [&](int j) {
#pragma unroll
        for (int i = 0; i < kOwn; ++i) next[i] = u + i * N < kStepKeys ? row_of(j, u + i * N) : ~0u;
      };
      look_up(0);
      bool ok = true;
      int pending = -1;  // slot whose cp.async copies are under way
      int sent = 0;      // behind the last slot filled, as the warp of the boxes counts them
      auto flush = [&](bool all) {
        if (pending < 0) return;
        if (all)
          cp_async_wait<0>();
        else
          cp_async_wait<1>();
        fence_async_proxy();
        tc::mbar_arrive(&ctl->kv_full[pending % Cfg::kStages]);
      };
      for (int j = 0; j < steps; ++j) {
        if (by_tma(j)) {
          if (u < 32) {
            const int pos = k_base + j * kStepKeys + box_key;
            for (int kind = 0; ok && kind < 2; ++kind) {
              const int i = 2 * j + kind, s = i % Cfg::kStages;
              if (i >= Cfg::kStages)
                ok = __all_sync(0xffffffffu, wait_for(&ctl->kv_empty[s],
                                                      (uint32_t)(i / Cfg::kStages - 1) & 1u, ctl));
              if (!ok) break;  // and on to the next step that all threads take, to say so
              if (lane == 0) {
                tc::mbar_arrive_expect_tx(&ctl->kv_full[s], Cfg::kKvBytes);
                mbar_arrive_many(&ctl->kv_full[s], N - 1);
              }
              __syncwarp();
              if (has_box)
                tma_load_page(ring + s * Cfg::kKvBytes + box_half * 16384 + box_key * 128, &map,
                              box_half * 64, kvh, page_slot(p, pos), page * 2 + kind,
                              &ctl->kv_full[s]);
              sent = i + 1;
            }
            page = page_of(j + 1);
          }
          if (pending >= 0) {
            flush(true);
            pending = -1;
          }
          if (j + 1 < steps && !by_tma(j + 1)) look_up(j + 1);
          continue;
        }
        ok = loaders_all<N>(ok);  // the rows of the step before are read
        if (!ok) break;
        const uint32_t* rws = ctl->rows;
#pragma unroll
        for (int i = 0; i < kOwn; ++i)
          if (u + i * N < kStepKeys) ctl->rows[u + i * N] = next[i];
        if (j + 1 < steps && !by_tma(j + 1))
          look_up(j + 1);
        else if (u < 32)
          page = page_of(j + 1);
#pragma unroll 1
        for (int kind = 0; kind < 2; ++kind) {
          const int i = 2 * j + kind;
          if (ok && i >= Cfg::kStages)
            ok = wait_for(&ctl->kv_empty[i % Cfg::kStages],
                          (uint32_t)(i / Cfg::kStages - 1) & 1u, ctl);
          ok = loaders_all<N>(ok);  // also: the step's rows are in place
          if (!ok) break;
          sent = i + 1;
          uint8_t* dst = ring + (i % Cfg::kStages) * Cfg::kKvBytes;
          if constexpr (!Q8) {
            constexpr int kChunks = D / 8;
#pragma unroll 4
            for (int x = u; x < kStepKeys * kChunks; x += N) {
              const int key = x / kChunks, c = x % kChunks;
              const uint32_t row = rws[key];
              const bool there = row != ~0u;
              const int64_t at = there ? (int64_t)row + kind * v_rows : 0;
              cp_async16(dst + tile_at(key, c), cache + at * (2 * D) + c * 16, there);
            }
            cp_async_commit();
            flush(false);  // the slot before this one has had a slot's time to arrive
            pending = i;
          } else {
            constexpr int kChunks = D / 16;  // 16 codes each
            constexpr int kEach = kStepKeys * kChunks / N;
            uint4 v[kEach];
            uint32_t ex[kEach];
#pragma unroll
            for (int x = 0; x < kEach; ++x) {
              const int key = (x * N + u) / kChunks, c = (x * N + u) % kChunks;
              const uint32_t row = rws[key];
              v[x] = make_uint4(0, 0, 0, 0);
              ex[x] = 127;
              if (row != ~0u) {
                const int64_t at = (int64_t)row + kind * v_rows;
                v[x] = ld_nc_v4(cache + at * D + c * 16);
                ex[x] = p.exponents[at];
              }
            }
#pragma unroll
            for (int x = 0; x < kEach; ++x) {
              const int key = (x * N + u) / kChunks, c = (x * N + u) % kChunks;
              const uint32_t w4[4] = {v[x].x, v[x].y, v[x].z, v[x].w};
              uint32_t o[8];
              M::dequantise16(w4, ex[x], o);
              *reinterpret_cast<uint4*>(dst + tile_at(key, 2 * c)) =
                  make_uint4(o[0], o[1], o[2], o[3]);
              *reinterpret_cast<uint4*>(dst + tile_at(key, 2 * c + 1)) =
                  make_uint4(o[4], o[5], o[6], o[7]);
            }
            fence_async_proxy();
            tc::mbar_arrive(&ctl->kv_full[i % Cfg::kStages]);
          }
        }
        if (!ok) break;
      }
      if constexpr (!Q8) {
        cp_async_wait<0>();
        if (ok) flush(true);
        // whatever ended the steps, no copy outlives the CTA; slots filled since then hold none
        for (int i = max(sent - Cfg::kStages, 0); u < 32 && i < sent; ++i)
          if (by_tma(i >> 1))
            tc::mbar_wait(&ctl->kv_full[i % Cfg::kStages], (uint32_t)(i / Cfg::kStages) & 1u,
                          kWaitLimitNs, nullptr);
      }
      if (!ok) tile_fault(ctl, fault);
    }
  }

  tc::tc_fence_before();
  __syncthreads();
  if (warp == 8) tc::tmem_dealloc(tmem, 512);
  if (w.splits == 1) return;

  // ---- the last piece of these rows to arrive joins them all --------------------
  // A piece whose waits ran out arrives too, so that the counter is zero again for the next call.
  if (!arrive_last(counters + (int64_t)w.tile * p.kv_heads + kvh, w.splits, &ctl->last)) return;
  if (*reinterpret_cast<volatile int*>(&ctl->abort)) return;
  if (warp >= 8) return;  // these gave their registers away
  join_pieces<T, 256, D, Q8, 256>(p, partial, partial_ml, w, kvh, group, rows,
                                  reinterpret_cast<float*>(ring),
                                  Cfg::kStages * Cfg::kKvBytes / 4);
}

// Tensor map of the cache as [2 * pages, page_size, kv_heads, D], boxes of `box`
// keys of one head: 64 dimensions, swizzled, of a 16-bit cache, a quantised
// one's whole rows as they are.
static int make_page_map(CUtensorMap* map, const Problem& p, CUtensorMapDataType type,
                         int64_t num_pages, int box, const char* what) {
  tc::EncodeTiledFn enc = tc::encode_tiled();
  if (!enc) return fail(PACE_ERR_CUDA, "%s: cuTensorMapEncodeTiled unavailable", what);
  const bool codes = type == CU_TENSOR_MAP_DATA_TYPE_UINT8;
  const cuuint64_t row = (cuuint64_t)p.head_dim * (codes ? 1 : 2);
  const cuuint64_t dims[4] = {(cuuint64_t)p.head_dim, (cuuint64_t)p.kv_heads,
                              (cuuint64_t)p.page_size, (cuuint64_t)(2 * num_pages)};
  const cuuint64_t strides[3] = {row, row * p.kv_heads, row * p.kv_heads * p.page_size};
  const cuuint32_t boxes[4] = {codes ? (cuuint32_t)p.head_dim : 64u, 1u, (cuuint32_t)box, 1u};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUresult r =
      enc(map, type, 4, const_cast<void*>(p.cache), dims, strides, boxes, estr,
          CU_TENSOR_MAP_INTERLEAVE_NONE,
          codes ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B,
          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(PACE_ERR_INVALID_ARGUMENT, "%s: tensor map rejected (CUresult %d)", what, (int)r);
  return PACE_OK;
}

template <typename T, int D, bool Q8>
static int run_tile(const Problem& p, int64_t num_pages, const Item* items, int num_items, float* partial, float2* ml,
                    int32_t* counters, int32_t* fault, int device, cudaStream_t stream,
                    const char* what) {
  using Cfg = TileCfg<D, Q8>;
  auto kernel = attention_tile_kernel<T, D, Q8>;
  cudaError_t err =
      ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), device, Cfg::kSmemBytes);
  if (err != cudaSuccess) return cuda_fail(err, what);
  // TMA where the pages allow it (8192 tokens: 528 us against 813 by 16-byte copies, quantised 706
  // against 881).  A box is a page's share of a 128-key step, and its 8-row swizzle groups have to
  // be the step's: pages of 8 to 128 keys that divide 128, or multiples of 128.
  CUtensorMap map{};
  int box = 0;
  if (p.page_size >= 8 && (128 % p.page_size == 0 || p.page_size % 128 == 0) &&
      num_pages < (1 << 30)) {
    box = p.page_size < 128 ? p.page_size : 128;
    const CUtensorMapDataType type = Q8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                     : std::is_same<T, __nv_bfloat16>::value
                                         ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                         : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const int st = make_page_map(&map, p, type, num_pages, box, what);
    if (st != PACE_OK) return st;
  }
  err = launch(kernel, dim3((unsigned)(num_items * p.kv_heads)), dim3(Cfg::kThreads),
               Cfg::kSmemBytes, stream, p, map, box, items, partial, ml, counters, fault);
  return err == cudaSuccess ? PACE_OK : cuda_fail(err, what);
}

int run_tile_rows(const Problem& p, int64_t num_pages, const Item* items, int num_items, float* partial, float2* ml,
                  int32_t* counters, int32_t* fault, bool bf16, int device, cudaStream_t stream,
                  const char* what) {
  auto pick = [&](auto t) -> int {
    using T = decltype(t);
    auto go = [&](auto f) {
      return f(p, num_pages, items, num_items, partial, ml, counters, fault, device, stream, what);
    };
    if (p.head_dim == 128)
      return p.exponents ? go(run_tile<T, 128, true>) : go(run_tile<T, 128, false>);
    return p.exponents ? go(run_tile<T, 64, true>) : go(run_tile<T, 64, false>);
  };
  return bf16 ? pick(__nv_bfloat16{}) : pick(__half{});
}

}  // namespace attn
}  // namespace pace
