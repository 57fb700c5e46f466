// Paged attention of few query rows: a request's new tokens times the query
// heads of one kv head, at most 16 rows (single tokens of grouped heads, short
// drafts).  Every key and value is read once for so few products that memory
// bounds it: the 16 x 8 x 16 matrix instructions of a warp are enough, and
// what counts is the bytes in flight.  64 single tokens of 32 heads over up to
// 8191 bf16 tokens each (1.2 GB) take 182 us, 6.5 TB/s, a copy's rate; over a
// quantised cache (597 MB) 166 us, 3.6 TB/s, where unpacking the codes bounds it
// (a single call alone: 147).  Distance bias adds 2 and 10 us.
//
// A CTA takes one piece of the plan (keys [kv_begin, kv_end) of one request)
// for one kv head.  Its four warps walk the keys in turns of KEYS each, every
// warp on its own: it copies its keys' K and V rows page by page into its own
// ring of STAGES slots (cp.async, no barrier between warps), multiplies them
// with the queries that sit in registers, and keeps the running maximum m, sum
// l and unnormalised output of its keys in registers, all fp32.  The warps'
// results are joined at the end:
//   M = max m_w,  o = sum_w 2^(m_w - M) o_w / sum_w 2^(m_w - M) l_w.
// Pieces of the same rows leave (m, l, o) in the workspace; the last to arrive
// joins them in the same way, in piece order, so results do not depend on the
// order of arrival.
//
// A quantised cache is copied as it is and unpacked between shared memory and
// the matrix instruction, which then works in fp16 whatever the query's type: a
// code moved to the top of 16 bits is its value times 2^-8 as fp16 holds it,
// subnormals included, and no multiplication touches it.  Every other word goes by
// the conversion instruction instead, which runs on another unit (all by it: 238 us
// for the 64 requests, all by shifts: 170, half and half: 166 then, 147 now).
// K's factor multiplies the scores.  V's factor 2^e goes into P: the output has a
// running maximum of its own, of score + e, and is built from 2^(score + e - it), so
// that the row's largest contribution is about 1 in fp16 whatever the factors are;
// the sum l keeps the maximum of the scores alone.  That holds for rows whose largest
// code is near 448, as the append makes them; where another cache's rows break it, the
// output shows it and the row is done again on the CUDA cores.  Queries are scaled by a power
// of two to the top of fp16's range: a bf16 query keeps all its bits down to 2^-29
// of its largest element.
#include "attention_mma.cuh"

namespace pace {
namespace attn {

constexpr int kFewWarps = 4;
constexpr float kLag = 8.f;  // in powers of two
// Over a quantised cache: the least size of an output, in units of its largest contribution's
// weight times one code, that its products in fp16 are trusted with.
constexpr float kLeastOutput = 32.f * 128;
// Exponents of V below this are those of zeros: 448 * 2^-100 * 2^-25 times any length is nothing.
constexpr float kFaintExponent = -100.f;

template <int D, bool Q8, int R>
struct FewTile {
  static constexpr int kKeys = D == 128 && !Q8 ? 16 : 32;  // of a warp's turn
  static constexpr int kRowBytes = Q8 ? D : 2 * D;
  static constexpr int kChunks = kRowBytes / 16;
  static constexpr int kKvBytes = kKeys * kRowBytes;
  // One row half of a quantised cache fits three CTAs an SM with two slots each (64 requests: 170
  // us, two CTAs with three slots 180); the others two CTAs with three.
  static constexpr int kCtas = Q8 && R == 1 ? 3 : 2;
  static constexpr int kStages = Q8 && R == 1 ? 2 : 3;
  static constexpr int kRingBytes = kStages * 2 * kKvBytes;
  static constexpr int kJoinBytes = 16 * D * 4;  // a warp's output, over its ring
  static constexpr int kWarpBytes = kRingBytes > kJoinBytes ? kRingBytes : kJoinBytes;
  // K's factors and V's exponents (both fp32) of the keys in the ring
  static constexpr int kFactorBytes = Q8 ? kStages * kKeys * 8 : 0;
  static constexpr int kSmemBytes = kFewWarps * (kWarpBytes + kFactorBytes) + kFewWarps * 32 * 4;
  // 16-byte chunk c of row r, placed so that eight rows' same chunk, and one
  // row's eight chunks, lie in different banks
  __device__ static __forceinline__ int at(int r, int c) {
    const int x = kChunks >= 8 ? (r & 7) : ((r >> 1) & 3);
    return r * kRowBytes + ((c ^ x) << 4);
  }
};

// A quantised word's two pairs of values as fp16: every other one by the
// conversion instruction, as they are, the rest by shifts, times 2^-8.  The two
// run on different units, neither of which alone keeps up with the memory.
__device__ __forceinline__ constexpr bool by_conversion(int n) { return n & 1; }
template <typename M>
__device__ __forceinline__ void unpack_by(bool conversion, uint32_t w, uint32_t& even,
                                          uint32_t& odd) {
  if (conversion) {
    const uint32_t x = __byte_perm(w, 0, 0x3120);
    even = e4m3x2_to_half2(x & 0xffffu);
    odd = e4m3x2_to_half2(x >> 16);
  } else {
    M::unpack_codes(w, even, odd);
  }
}

// The larger of two, NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// cap * tanh(x / cap) as a difference, off by about cap * 2^-22.
__device__ __forceinline__ float cap_score(float x, float cap, float cap_in) {
  return cap - 2.f * cap * rcp_approx(1.f + exp2_approx(x * cap_in));
}
// Scores well within a cap larger than this would not bear that.  Up to a quarter
// of it they take four terms of the series of tanh(u) / u instead (the fifth is
// 3.3e-7 there), whose error goes with the score.  Choosing in the one kernel for
// all caps took 64 requests over a quantised cache without any from 163 to 189 us.
constexpr float kLargeCap = 512.f;
__device__ __forceinline__ float large_cap_score(float x, float cap, float inv_cap,
                                                 float cap_in) {
  const float u = x * inv_cap, z = u * u;
  const float near = x * fmaf(z, fmaf(z, fmaf(z, -17.f / 315.f, 2.f / 15.f), -1.f / 3.f), 1.f);
  return fabsf(u) <= 0.25f ? near : cap_score(x, cap, cap_in);
}

// R: 1 where the rows fit the matrix instruction's first eight, else 2.  LARGE:
// the cap is a large one.
template <typename T, int D, bool Q8, int R, bool LARGE>
__global__ void __launch_bounds__(kFewWarps * 32, FewTile<D, Q8, R>::kCtas)
    attention_few_kernel(const Problem p, const Item* items, float* partial,
                         float2* partial_ml, int32_t* counters, bool q_even, bool beside) {
  using Tile = FewTile<D, Q8, R>;
  using M = Mma<std::conditional_t<Q8, __half, T>>;
  // what P, and with it the sum, is scaled up by; over a quantised cache P alone, see base_o
  constexpr float kUp = !Q8 && std::is_same<T, __half>::value ? kHeadroom : 0.f;
  constexpr int KEYS = Tile::kKeys, NT = KEYS / 8, KB = D / 16, STAGES = Tile::kStages;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint32_t faint;  // rows to be done again
  if (threadIdx.x == 0) faint = 0;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  const int kvh = blockIdx.x % p.kv_heads;
  const int group = p.heads / p.kv_heads;
  uint8_t* ring = smem + warp * Tile::kWarpBytes;
  float* factors = reinterpret_cast<float*>(smem + kFewWarps * Tile::kWarpBytes +
                                            warp * Tile::kFactorBytes);
  float* v_exps = factors + Tile::kStages * KEYS;
  float* join_ml = reinterpret_cast<float*>(
      smem + kFewWarps * (Tile::kWarpBytes + Tile::kFactorBytes));  // [warp][16][m, l]
  // `beside`: the kernel before this one in the stream is the tile kernel of the same call, which
  // this one reads nothing of and which let it start only when all before both was complete.  It
  // then waits for that kernel at its end, for the sake of what comes after.
  pdl_launch_dependents();
  if (!beside) pdl_wait();
  const Item w = items[blockIdx.x / p.kv_heads];  // not earlier: a kernel may have written the plan
  const int rows = w.ntok * group;

  // ---- the ring: its first copies are under way while the queries are fetched --------
  const uint8_t* cache = static_cast<const uint8_t*>(p.cache);
  const int64_t v_rows = (int64_t)p.page_size * p.kv_heads, v_bytes = v_rows * Tile::kRowBytes;
  const int begin = w.kv_begin + warp * KEYS;
  const int steps = begin < w.kv_end ? (w.kv_end - begin + kFewWarps * KEYS - 1) / (kFewWarps * KEYS) : 0;
  const int my_key = lane % KEYS;
  auto page_of = [&](int step) -> int {
    const int j = begin + step * kFewWarps * KEYS + my_key;
    return step < steps && j < w.kv_end ? p.kv_indices[w.page_base + page_number(p, j)] : -1;
  };
  uint32_t k_ex = 0, v_ex = 0;  // exponents of this lane's key of the step issued last
  auto issue = [&](int step, int page) {
    // row number (of the whole cache, K part) of this lane's key; ~0: none
    uint32_t row = ~0u;
    if (page >= 0) {
      const int j = begin + step * kFewWarps * KEYS + my_key;
      row = (uint32_t)(((int64_t)page * 2 * p.page_size + page_slot(p, j)) * p.kv_heads + kvh);
    }
    uint8_t* slot = ring + (step % STAGES) * 2 * Tile::kKvBytes;
#pragma unroll
    for (int i = 0; i < KEYS * Tile::kChunks / 32; ++i) {
      const int r = (i * 32 + lane) / Tile::kChunks, ch = (i * 32 + lane) % Tile::kChunks;
      const uint32_t src = __shfl_sync(0xffffffffu, row, r);
      const bool there = src != ~0u;
      const uint8_t* k = cache + (there ? (int64_t)src * Tile::kRowBytes + ch * 16 : 0);
      const int at = Tile::at(r, ch);
      cp_async16(slot + at, k, there);
      cp_async16(slot + Tile::kKvBytes + at, k + (there ? v_bytes : 0), there);
    }
    if constexpr (Q8) {
      k_ex = v_ex = 0;
      if (row != ~0u) {
        k_ex = p.exponents[row];
        v_ex = p.exponents[row + v_rows];
      }
    }
  };
  auto put_factors = [&](int step) {
    if constexpr (Q8) {
      factors[(step % STAGES) * KEYS + lane] = exponent_factor(k_ex);
      v_exps[(step % STAGES) * KEYS + lane] =
          v_ex == (uint32_t)kNanExponent ? exponent_factor(kNanExponent) : (float)v_ex - 127.f;
    }
  };

  uint32_t k_first[STAGES - 1], v_first[STAGES - 1];
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) {
    issue(s, page_of(s));
    cp_async_commit();
    k_first[s] = k_ex;
    v_first[s] = v_ex;
  }
  int page = page_of(STAGES - 1);

  // ---- rows g and g + 8 of this thread: visible keys, slope, queries --------
  int lo[R], hi[R], pos[R];
  float slope[R];
  const uint64_t* bits[R] = {};
  int all_lo = 0, all_hi = INT32_MAX;  // keys that every row sees
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = g + 8 * i;
    lo[i] = 0;
    hi[i] = INT32_MAX;
    pos[i] = 0;
    slope[i] = 0.f;
    if (r < rows) {
      const int tok = w.tok0 + r / group;
      const TokenInfo t = p.tokens[tok];
      lo[i] = t.lo;
      hi[i] = t.hi;
      pos[i] = t.pos;
      if (p.slopes) slope[i] = p.slopes[kvh * group + r % group] * kLog2e;
      if (p.tree_mask) bits[i] = p.tree_mask + (int64_t)tok * p.tree_words;
      all_lo = max(all_lo, lo[i]);
      all_hi = min(all_hi, hi[i]);
    }
  }
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) {
    all_lo = max(all_lo, __shfl_xor_sync(0xffffffffu, all_lo, o));
    all_hi = min(all_hi, __shfl_xor_sync(0xffffffffu, all_hi, o));
  }
  uint32_t qf[KB][4];
  {
    const T* q[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = g + 8 * i;
      q[i] = r < rows ? static_cast<const T*>(p.query) + (int64_t)(w.tok0 + r / group) * p.q_stride +
                            (int64_t)(kvh * group + r % group) * D
                      : nullptr;
    }
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const T* row = (i & 1) < R ? q[i & 1] : nullptr;
        // the two dimensions of this register: those that the keys' register of the same
        // index holds (a quantised key's registers hold bytes 0, 2 and 1, 3 of four)
        const int d0 = Q8 ? kb * 16 + 4 * c + (i >> 1) : kb * 16 + 2 * c + 8 * (i >> 1);
        if (!row)
          qf[kb][i] = 0;
        else if (!Q8 && q_even)
          qf[kb][i] = *reinterpret_cast<const uint32_t*>(row + d0);
        else
          qf[kb][i] = Mma<T>::pair(row[d0], row[d0 + (Q8 ? 2 : 1)]);
      }
  }
  float row_scale[R];
#pragma unroll
  for (int i = 0; i < R; ++i) row_scale[i] = p.scale * kLog2e;
  if constexpr (Q8) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      float top = 0.f;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int k = i; k < 4; k += 2) {
          const float2 x = Mma<T>::floats(qf[kb][k]);
          top = fmaxf(top, fmaxf(fabsf(x.x), fabsf(x.y)));
        }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // the power of two that brings `top` to 2^14 .. 2^15
      const uint32_t up = min(268u - (__float_as_uint(top) >> 23), 254u);
      const float f = __uint_as_float(up << 23);
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int k = i; k < 4; k += 2) {
          const float2 x = Mma<T>::floats(qf[kb][k]);
          qf[kb][k] = M::pack(x.x * f, x.y * f);
        }
      row_scale[i] *= 1.f / f;
    }
  }

#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) {
    k_ex = k_first[s];
    v_ex = v_first[s];
    put_factors(s);
  }
  float o[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
  float m[R], l[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
  }
  // over a quantised cache: the running maximum of score + V's exponent; O is in units of 2^mo
  float mo[R];
#pragma unroll
  for (int i = 0; i < R; ++i) mo[i] = -INFINITY;
  const float cap2 = p.cap * kLog2e, cap_in = p.cap > 0.f ? 2.f / p.cap : 0.f;
  const float inv_cap2 = LARGE ? 1.f / cap2 : 0.f;

  for (int step = 0; step < steps; ++step) {
    if (step > 0) put_factors(step + STAGES - 2);  // their loads had a step's time
    issue(step + STAGES - 1, page);
    cp_async_commit();
    page = page_of(step + STAGES);
    cp_async_wait<STAGES - 1>();
    __syncwarp();
    const uint8_t* ks = ring + (step % STAGES) * 2 * Tile::kKvBytes;
    const uint8_t* vs = ks + Tile::kKvBytes;
    const float* kf = factors + (step % STAGES) * KEYS;
    const float* ve = v_exps + (step % STAGES) * KEYS;
    // ---- S = Q K^T ------------------------------------------------------------
    float s[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      if constexpr (Q8) {
        uint32_t r[4];
        ldmatrix4(r, ks + Tile::at(lane, kb));
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          uint32_t b0, b1;
          unpack_by<M>(by_conversion(n), r[n], b0, b1);
          M::mma(s[n], qf[kb], b0, b1);
        }
      } else {
#pragma unroll
        for (int n = 0; n < NT; n += 2) {
          uint32_t r[4];
          ldmatrix4(r, ks + Tile::at(n * 8 + (lane >> 4) * 8 + (lane & 7), 2 * kb + ((lane >> 3) & 1)));
          M::mma(s[n], qf[kb], r[0], r[1]);
          M::mma(s[n + 1], qf[kb], r[2], r[3]);
        }
      }
    }
    // ---- scores in powers of two, masks ---------------------------------------
    const int j0 = begin + step * kFewWarps * KEYS;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float2 f = make_float2(1.f, 1.f);
      if constexpr (Q8) {
        f = *reinterpret_cast<const float2*>(kf + n * 8 + 2 * c);
        if (!by_conversion(n)) {  // the shifted codes' 2^-8
          f.x *= 256.f;
          f.y *= 256.f;
        }
      }
#pragma unroll
      for (int e = 0; e < 2 * R; ++e) {
        float x = s[n][e] * row_scale[e >> 1];
        if constexpr (Q8) x *= e & 1 ? f.y : f.x;
        if constexpr (LARGE)
          x = large_cap_score(x, cap2, inv_cap2, cap_in);
        else if (p.cap > 0.f)
          x = cap_score(x, cap2, cap_in);
        s[n][e] = x;
      }
    }
    if (p.slopes) {
#pragma unroll
      for (int i = 0; i < R; ++i) {
        // from the row's token to the thread's first key; it is before the token in most steps,
        // where the bias rises by the slope from key to key
        const float away = (float)(pos[i] - j0 - 2 * c);
        const float first = -slope[i] * away;
        const bool before = away >= (float)KEYS;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float k = (float)(n * 8 + e);
            s[n][2 * i + e] += before ? fmaf(slope[i], k, first) : -slope[i] * fabsf(away - k);
          }
      }
    }
    if (j0 < all_lo || j0 + KEYS > min(all_hi, w.kv_end)) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2 * R; ++e) {
          const int j = j0 + n * 8 + 2 * c + (e & 1), i = e >> 1;
          bool see = j >= lo[i] && j < hi[i] && j < w.kv_end;
          if (bits[i] && j >= hi[i]) see = j < min(pos[i], w.kv_end) && tree_bit(bits[i], j - hi[i]);
          if (!see) s[n][e] = -INFINITY;
        }
    }
    // ---- running maximum and sum: the maximum may lag by 2^kLag, so that most steps
    // need neither the row's maximum, which its lanes share by shuffles, nor a new scale
    float most[R], most_o[R];
    bool rise = false;
    float2 v_e[NT];
    if constexpr (Q8) {
#pragma unroll
      for (int n = 0; n < NT; ++n) v_e[n] = *reinterpret_cast<const float2*>(ve + n * 8 + 2 * c);
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      most[i] = most_o[i] = -INFINITY;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        most[i] = fmaxf(most[i], fmaxf(s[n][2 * i], s[n][2 * i + 1]));
        if constexpr (Q8)
          most_o[i] = fmaxf(most_o[i], fmaxf(s[n][2 * i] + v_e[n].x, s[n][2 * i + 1] + v_e[n].y));
      }
      rise |= most[i] > m[i] + kLag || (m[i] == -INFINITY && most[i] > m[i]);
      if constexpr (Q8)
        rise |= most_o[i] > mo[i] + kLag || (mo[i] == -INFINITY && most_o[i] > mo[i]);
    }
    if (__any_sync(0xffffffffu, rise)) {
      auto raise = [](float& old, float t) {  // to the row's maximum; returns what that scales by
        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 1));
        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 2));
        const float now = fmaxf(old, t);
        const float f = exp2_approx(old - (now == -INFINITY ? 0.f : now));  // 0 while old is -inf
        old = now;
        return f;
      };
#pragma unroll
      for (int i = 0; i < R; ++i) {
        float f = raise(m[i], most[i]);
        l[i] *= f;
        if constexpr (Q8) f = raise(mo[i], most_o[i]);
#pragma unroll
        for (int n = 0; n < D / 8; ++n) {
          o[n][2 * i] *= f;
          o[n][2 * i + 1] *= f;
        }
      }
    }
    float base[R], base_o[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      base[i] = m[i] == -INFINITY ? 0.f : m[i] - kUp;
      base_o[i] = mo[i] == -INFINITY ? 0.f : mo[i] - kHeadroom;
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2 * R; ++e) {
        const float y = s[n][e];
        const float x = exp2_approx(y - base[e >> 1]);
        l[e >> 1] += x;
        if constexpr (Q8) {
          // a key that the row does not see stays 0 whatever its row holds
          const float z = y + ((e & 1 ? v_e[n].y : v_e[n].x) - base_o[e >> 1]);
          s[n][e] = y == -INFINITY ? 0.f : exp2_approx(z);
        } else {
          s[n][e] = x;
        }
      }
    // ---- O += P V; P is rounded to T, the one rounding before the output's ----
#pragma unroll
    for (int kg = 0; kg < NT / 2; ++kg) {
      uint32_t a[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        a[i] = 0;
        if ((i & 1) >= R) continue;
        const float x = s[2 * kg + (i >> 1)][2 * (i & 1)], y = s[2 * kg + (i >> 1)][2 * (i & 1) + 1];
        a[i] = M::pack(x, y);
      }
      if constexpr (Q8) {
#pragma unroll
        for (int ch = 0; ch < D / 16; ch += 2) {
          uint32_t r[4];
          // keys kg * 16 + 0-7, 8-15 of chunks ch, ch + 1: two keys' pairs of dimensions
          ldmatrix4_trans(r, vs + Tile::at(kg * 16 + (lane & 15), ch + (lane >> 4)));
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t e0, d0, e1, d1;
            unpack_by<M>(by_conversion(ch + h), r[2 * h], e0, d0);
            unpack_by<M>(by_conversion(ch + h), r[2 * h + 1], e1, d1);
            M::mma(o[2 * (ch + h)], a, e0, e1);
            M::mma(o[2 * (ch + h) + 1], a, d0, d1);
          }
        }
      } else {
#pragma unroll
        for (int ch = 0; ch < D / 8; ch += 2) {
          uint32_t r[4];
          ldmatrix4_trans(r, vs + Tile::at(kg * 16 + (lane & 15), ch + (lane >> 4)));
          M::mma(o[ch], a, r[0], r[1]);
          M::mma(o[ch + 1], a, r[2], r[3]);
        }
      }
    }
    __syncwarp();  // the slot is free for the copies of the next turn
  }
  cp_async_wait<0>();
  __syncthreads();

  // ---- join the warps ----------------------------------------------------------
#pragma unroll
  for (int i = 0; i < R; ++i) {
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    const int r = g + 8 * i;
    if constexpr (Q8) {
      // The key that set the output's maximum adds its weight of 1 times its largest code, 224 or
      // more of a row as the append writes it.  An output that stays far below had its maximum
      // set by a row that adds little or nothing (zeros under a large exponent), and what counts
      // may have been lost below fp16.  Not where that row's factor is next to nothing itself, as
      // the append gives it to zeros: then so is all that is lost.  NaN is left as it is.
      float top = 0.f;
#pragma unroll
      for (int n = 0; n < D / 8; ++n) {
        const float up = by_conversion(n >> 1) ? 1.f : 256.f;
        top = max_nan(top, max_nan(fabsf(o[n][2 * i]), fabsf(o[n][2 * i + 1])) * up);
      }
      top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 2));
      if (c == 0 && r < rows && mo[i] > m[i] + kFaintExponent && top < kLeastOutput)
        atomicOr(&faint, 1u << r);
    }
    if (r < rows) {
      if (c == 0) {
        join_ml[(warp * 16 + r) * 2] = m[i] - kUp;
        join_ml[(warp * 16 + r) * 2 + 1] = l[i];
      }
      float* dst = reinterpret_cast<float*>(ring) + r * D;
      // in the joined output's units, 2^m
      const float unit =
          Q8 ? (mo[i] == -INFINITY ? 0.f : exp2_approx(mo[i] - kHeadroom - m[i])) : 1.f;
#pragma unroll
      for (int n = 0; n < D / 8; ++n) {
        const float up = Q8 && !by_conversion(n >> 1) ? 256.f : 1.f;
        const int d = Q8 ? (n >> 1) * 16 + 4 * c + (n & 1) : n * 8 + 2 * c;
        dst[d] = o[n][2 * i] * up * unit;
        dst[d + (Q8 ? 2 : 1)] = o[n][2 * i + 1] * up * unit;
      }
    }
  }
  __syncthreads();
  constexpr int V4 = D / 4;
  const int64_t slot = (int64_t)(w.slot + w.split) * p.kv_heads + kvh;
  const uint32_t redo = Q8 ? *reinterpret_cast<volatile uint32_t*>(&faint) : 0;
  // whole warps stay in the loop, for redo_rows
  for (int u = threadIdx.x; (u & ~31) < rows * V4; u += kFewWarps * 32) {
    const int r = u / V4, d = (u - r * V4) * 4;
    bool fine = true;
    if (u < rows * V4) {
      float mm = -INFINITY;
#pragma unroll
      for (int k = 0; k < kFewWarps; ++k) mm = fmaxf(mm, join_ml[(k * 16 + r) * 2]);
      const float b = mm == -INFINITY ? 0.f : mm;
      float sum = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < kFewWarps; ++k) {
        const float f = exp2_approx(join_ml[(k * 16 + r) * 2] - b);
        sum += f * join_ml[(k * 16 + r) * 2 + 1];
        const float4 x = *reinterpret_cast<const float4*>(smem + k * Tile::kWarpBytes + (r * D + d) * 4);
        v[0] += f * x.x;
        v[1] += f * x.y;
        v[2] += f * x.z;
        v[3] += f * x.w;
      }
      if (w.splits == 1) {
        fine = write_out<T>(p, w.tok0 + r / group, kvh * group + r % group, d, v, mm, sum);
        fine |= !w.mixed;
      } else {
        __stcg(reinterpret_cast<float4*>(partial + (slot * 16 + r) * D + d),
               make_float4(v[0], v[1], v[2], v[3]));
        // the sign of the sum tells the piece that joins
        if (d == 0) __stcg(partial_ml + slot * 16 + r, make_float2(mm, redo >> r & 1 ? -sum : sum));
      }
    }
    if (w.splits == 1 && (w.mixed || redo))
      redo_rows<T, D, Q8>(p, w, kvh, group, r, fine, u < rows * V4 && (redo >> r & 1));
  }
  if (w.splits == 1) {
    if (beside) pdl_wait();
    return;
  }

  // ---- the last piece of these rows to arrive joins them all --------------------
  __shared__ bool last;
  if (arrive_last(counters + (int64_t)w.tile * p.kv_heads + kvh, w.splits, &last))
    join_pieces<T, 16, D, Q8, kFewWarps * 32>(p, partial, partial_ml, w, kvh, group, rows,
                                              reinterpret_cast<float*>(smem),
                                              kFewWarps * Tile::kWarpBytes / 4);
  if (beside) pdl_wait();
}

template <typename T, int D, bool Q8, int R, bool LARGE>
static int run_few_r(const Problem& p, const Item* items, int num_items, float* partial, float2* ml,
                     int32_t* counters, bool beside, int device, cudaStream_t stream,
                     const char* what) {
  using Tile = FewTile<D, Q8, R>;
  auto kernel = attention_few_kernel<T, D, Q8, R, LARGE>;
  cudaError_t err =
      ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), device, Tile::kSmemBytes);
  if (err != cudaSuccess) return cuda_fail(err, what);
  const bool even = (reinterpret_cast<uintptr_t>(p.query) & 3) == 0 && p.q_stride % 2 == 0;
  err = launch(kernel, dim3((unsigned)(num_items * p.kv_heads)), dim3(kFewWarps * 32),
               Tile::kSmemBytes, stream, p, items, partial, ml, counters, even, beside);
  return err == cudaSuccess ? PACE_OK : cuda_fail(err, what);
}

template <typename T, int D, bool Q8>
static int run_few(const Problem& p, int max_rows, const Item* items, int num_items, float* partial,
                   float2* ml, int32_t* counters, bool beside, int device, cudaStream_t stream,
                   const char* what) {
  auto go = [&](auto f) {
    return f(p, items, num_items, partial, ml, counters, beside, device, stream, what);
  };
  if (p.cap > kLargeCap) return go(run_few_r<T, D, Q8, 2, true>);
  return max_rows <= 8 ? go(run_few_r<T, D, Q8, 1, false>) : go(run_few_r<T, D, Q8, 2, false>);
}

int run_few_rows(const Problem& p, int max_rows, const Item* items, int num_items, float* partial,
                 float2* ml, int32_t* counters, bool beside, bool bf16, int device,
                 cudaStream_t stream, const char* what) {
  auto pick = [&](auto t) -> int {
    using T = decltype(t);
    auto go = [&](auto f) {
      return f(p, max_rows, items, num_items, partial, ml, counters, beside, device, stream, what);
    };
    if (p.head_dim == 128) return p.exponents ? go(run_few<T, 128, true>) : go(run_few<T, 128, false>);
    return p.exponents ? go(run_few<T, 64, true>) : go(run_few<T, 64, false>);
  };
  return bf16 ? pick(__nv_bfloat16{}) : pick(__half{});
}

}  // namespace attn
}  // namespace pace
