// Attention with scores by rule, forward pass on tcgen05 tensor cores, for 16-bit heads of up to 128 (multiples of 8; narrower ones are filled
// with zeros by the tile copies).  A CTA has one tile of 128 rows: four warps on the scores, a thread a row, whose 128 scores of a tile stay in
// registers from their one read of TMEM to their exponentials; a TMA warp; an MMA warp.  P is handed over through TMEM, O stays there and
// is rescaled only when a maximum grows by more than 2^8.  Two CTAs share an SM (256 columns of TMEM and 96 KB each): one's exponentials run while
// the other's products do, and the start and end of one hide behind the middle of the other.  One CTA of two row tiles an SM, which
// reads keys and values once for both, took 400 us where this takes 359 to 375 (capped, 2 x 4096 x 32/8 x 128; uncapped 295; the longer under the power
// cap of a long run), with an issuer a row tile 426: the tiles fell into step; products of 64 keys at a time run at half their rate.
//
// What the rules add:
//   tiles       the flags of every tile of 128 keys (left out / looked at / whole) are worked out once, before the roles part; all of
//               them walk over the same list, so that what no row of a tile sees costs nothing.  A tile that is cut costs more than a whole one, most
//               of all by documents, whose ids are compared pair by pair: 16 x 1024 x 12 x 64 82 us causal, 73 in a window of 300, 75 with documents of 300 on
//               average, of which 59 % of the tiles are looked at
//   cap         tanh as a polynomial on the FMA pipe while no score of the warp is beyond three quarters of the cap; where a tile is whole and has no slopes, its last
//               product and the subtraction of the maximum are one multiply-add
//   distance    where all keys lie behind the rows, slope * |i - j| is slope * e of the key's place in the tile, from a table, and a number of the row
//   masks       128 bits a row, in tiles that are not whole; segments by comparing with ids that the warp loads once and hands around
// A row that sees nothing keeps a maximum of -inf and becomes zero.
//
// What bounds it: an exponential a score, 2048 cycles a pair of tiles on the special-function pipe, and products of about 2800 (operands from
// shared memory) at the least; no pipe is busy for more than half of the time, and what lasts is a tile's chain of product, scores, exponentials and product, of
// which the two CTAs overlap a part.  A share of the exponentials as a polynomial on the FMA pipe made it slower: with two warps a scheduler its longer chains show.
//
// For training the CTA stores L = max + log2(sum) of each row, and P goes to the product with the values in two parts, itself in 16 bits and
// what that rounding lost (the columns are free: P takes half of the scores').  O is then exact to float32 but for its own rounding, and what
// that lost is stored beside it (`lo`): the gradient needs sum_d dO O to more than eight bits.  With P in one part, gradients were 1.6 to 1.75
// times as far off as plain float32 rounded once, now 1.4; it costs 5 % of a training step.
#include "attention_rules_sm100.cuh"

namespace {
using namespace kbrules;

template <int D>
struct FwdCfg {
  static constexpr int CH = D / 64;
  static constexpr int TILE = CH * 16384;
  static constexpr int RING = D == 128 ? 2 : 4;
  static constexpr int BARS = (1 + RING) * TILE;
  static constexpr int RAMP = BARS + 256;  // slope * e of the head, e = 0 .. 127
  static constexpr int FLAGS = RAMP + 512;
  static constexpr int SMEM = FLAGS;  // and a byte a tile of keys
  static constexpr uint32_t TMEM_COLS = 256;
  static constexpr int THREADS_ = 192;  // four warps on the scores, one for copies, one for products
};
constexpr float RESCALE = 8.f;

// Ties registers that tcgen05.ld fills to the wait before it, so that nothing reads them earlier.
__device__ __forceinline__ void loaded(float (&x)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int e = 0; e < 32; e += 8)
    asm volatile("" : "+f"(x[e]), "+f"(x[e + 1]), "+f"(x[e + 2]), "+f"(x[e + 3]), "+f"(x[e + 4]), "+f"(x[e + 5]), "+f"(x[e + 6]), "+f"(x[e + 7]));
}
__device__ __forceinline__ void max32(float (&m)[4], const float (&x)[32]) {
#pragma unroll
  for (int e = 0; e < 32; e += 8)
#pragma unroll
    for (int u = 0; u < 4; ++u) m[u] = max3_nan(m[u], x[e + u], x[e + 4 + u]);
}
// Maximum of 32 products, and their largest magnitude, where they are wanted.
__device__ __forceinline__ void extremes(const float (&x)[32], float (&m)[4], float& top, bool want_max, bool want_top) {
  if (want_max) max32(m, x);
  if (want_top) {
#pragma unroll
    for (int e = 0; e < 32; e += 2) top = fmaxf(fmaxf(top, fabsf(x[e])), fabsf(x[e + 1]));
  }
}
// From products to scores, their masks and their maximum: what no shorter way takes.  Returns what has to be added to the scores: where all of
// the warp's keys lie behind its rows (`behind`), slope * |i - j| is slope * e of the key's place in the tile less a number of the row.
__device__ __forceinline__ float finish_scores(float (&x)[4][32], uint32_t at, float (&m)[4], bool cap, const Cap& c_, float post, float slope, int from, const float* ramp, bool whole,
                                               const uint32_t (&keep)[4], bool behind) {
  if (cap) {
    float top = 0.f;
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int e = 0; e < 32; e += 2) top = fmaxf(fmaxf(top, fabsf(x[c][e])), fabsf(x[c][e + 1]));
    const uint64_t pre2 = both(c_.pre);
    top *= fabsf(c_.pre);  // what is masked has a say too: at worst, the longest form
    if (!__any_sync(0xffffffffu, top > 0.5f)) {
      const uint64_t a0 = both(c_.near[0]), a1 = both(c_.near[1]), a2 = both(c_.near[2]), a3 = both(c_.near[3]);
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const uint64_t v = mul_f32x2(pack_f32x2(x[c][e], x[c][e + 1]), pre2), u = mul_f32x2(v, v);
          unpack_f32x2(mul_f32x2(fma_f32x2(fma_f32x2(fma_f32x2(a3, u, a2), u, a1), u, a0), v), x[c][e], x[c][e + 1]);
        }
    } else if (!__any_sync(0xffffffffu, top > 1.f)) {
      const uint64_t a0 = both(c_.far[0]), a1 = both(c_.far[1]), a2 = both(c_.far[2]), a3 = both(c_.far[3]), a4 = both(c_.far[4]), a5 = both(c_.far[5]);
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const uint64_t v = mul_f32x2(pack_f32x2(x[c][e], x[c][e + 1]), pre2), u = mul_f32x2(v, v);
          unpack_f32x2(mul_f32x2(fma_f32x2(fma_f32x2(fma_f32x2(fma_f32x2(fma_f32x2(a5, u, a4), u, a3), u, a2), u, a1), u, a0), v), x[c][e], x[c][e + 1]);
        }
    } else {  // seldom: a loop through TMEM, for the size of the code
#pragma unroll 1
      for (int c = 0; c < 8; ++c) {
        uint32_t y[16];
        tmem_ld16(at + (uint32_t)(c * 16), y);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
        for (int e = 0; e < 16; ++e) y[e] = __float_as_uint(tanh_any(__uint_as_float(y[e]) * c_.pre) * c_.post);
        tmem_st16(at + (uint32_t)(c * 16), y);
      }
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        tmem_ld32(at + 32u * c, reinterpret_cast<uint32_t*>(x[c]));
        loaded(x[c]);
      }
    }
  }
  float offset = 0.f;
  const uint64_t post2 = both(cap ? 1.f : post);
  if (slope != 0.f && behind) {
    offset = -slope * (float)from;
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int e = 0; e < 32; e += 4) {
        const ulonglong2 r = *reinterpret_cast<const ulonglong2*>(ramp + 32 * c + e);
        unpack_f32x2(fma_f32x2(pack_f32x2(x[c][e], x[c][e + 1]), post2, r.x), x[c][e], x[c][e + 1]);
        unpack_f32x2(fma_f32x2(pack_f32x2(x[c][e + 2], x[c][e + 3]), post2, r.y), x[c][e + 2], x[c][e + 3]);
      }
  } else if (slope != 0.f) {
    const float first = (float)from, step = cap ? 1.f : post;
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int e = 0; e < 32; ++e) x[c][e] = fmaf(-slope, fabsf(first - (float)(32 * c + e)), x[c][e] * step);
  } else if (!cap && post != 1.f) {
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int e = 0; e < 32; e += 2) unpack_f32x2(mul_f32x2(pack_f32x2(x[c][e], x[c][e + 1]), post2), x[c][e], x[c][e + 1]);
  }
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    if (!whole) {
#pragma unroll
      for (int e = 0; e < 32; ++e)
        if (!(keep[c] >> e & 1u)) x[c][e] = -INFINITY;
    }
    max32(m, x[c]);
  }
  return offset;
}
// P of 32 scores in 16 bits, and its sum.  score2(a pair) -> their exponents.  TRAIN: what rounding P lost follows 64 columns further, for a product of its own.
template <typename T, bool TRAIN, typename F>
__device__ __forceinline__ void exponentials(const float (&x)[32], uint32_t to, uint64_t (&l2)[2], F score2) {
  uint32_t w[16], lost[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    float x0, x1;
    unpack_f32x2(score2(pack_f32x2(x[2 * e], x[2 * e + 1])), x0, x1);
    x0 = ex2(x0);
    x1 = ex2(x1);
    w[e] = pack_16<T>(x0, x1);
    l2[e & 1] = add_f32x2(l2[e & 1], pack_f32x2(x0, x1));
    if (TRAIN) {
      float r0, r1;
      unpack_16<T>(w[e], r0, r1);
      lost[e] = pack_16<T>(x0 - r0, x1 - r1);
    }
  }
  tmem_st16(to, w);
  if (TRAIN) tmem_st16(to + 64u, lost);
}

template <typename T, int D, bool TRAIN>
__global__ void __launch_bounds__(FwdCfg<D>::THREADS_, 2)
rules_fwd_sm100(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                const Rules p, const Cap c_, T* o, T* lo_out, float* lse, int pitch, int* err) {
  using C = FwdCfg<D>;
  constexpr int TILE = C::TILE, RING = C::RING;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t base = smem_u32(smem_raw);
  if (base & 1023u) {
    if (threadIdx.x == 0 && err) atomicExch(err, 40);
    return;
  }
  const uint32_t sQ = base, sKV = sQ + TILE, bar_base = base + C::BARS;
  uint8_t* flags = smem_raw + C::FLAGS;  // of key tile first + n
  const uint32_t q_bar = bar_base;
  auto kv_full = [&](int s) { return bar_base + 8u * (1 + s); };
  auto kv_empty = [&](int s) { return bar_base + 8u * (1 + RING + s); };
  const uint32_t s_full = bar_base + 8u * (1 + 2 * RING), o_done = s_full + 8u;
  auto p_ready = [&](int u) { return s_full + 16u + 8u * u; };  // u = 0: of the first 96 keys, 1: of all
  constexpr int N_BARS = 5 + 2 * RING;
  static_assert(N_BARS * 8 + 8 <= 256, "barrier area");
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem_raw + C::BARS + N_BARS * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int groups = p.H * p.B, n_q = (p.Tq + BLK - 1) / BLK;
  const int q0 = (n_q - 1 - (int)(blockIdx.x / groups)) * BLK;  // the longest rows of a causal mask first
  const int h = (int)(blockIdx.x % groups) % p.H, b = (int)(blockIdx.x % groups) / p.H;
  const int hkv = h / (p.H / p.Hkv);
  const int prefix = prefix_of(p, b);
  int first, last;  // tiles of keys
  keys_of_rows(p, q0, min(q0 + BLK, p.Tq) - 1, prefix, first, last);
  first /= BLK;
  last = last < 0 ? -1 : last / BLK;
  for (int n = threadIdx.x; first + n <= last; n += C::THREADS_) flags[n] = (uint8_t)tile_flags(p, b, q0, (first + n) * BLK, prefix);
  const int end = last - first + 1;
  auto next = [&](int n) {  // the next tile that any of the rows needs, `end` if there is none
    do ++n;
    while (n < end && !(flags[n] & NEEDED));
    return n;
  };

  if (threadIdx.x < 128 && p.slopes != nullptr) reinterpret_cast<float*>(smem_raw + C::RAMP)[threadIdx.x] = score_of(p, h).slope * (float)threadIdx.x;
  if (threadIdx.x == 0) {
    mbar_init(q_bar, 1);
    for (int s = 0; s < RING; ++s) {
      mbar_init(kv_full(s), 1);
      mbar_init(kv_empty(s), 1);
    }
    mbar_init(s_full, 1);
    mbar_init(o_done, 1);
    mbar_init(p_ready(0), 4);
    mbar_init(p_ready(1), 4);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 5) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32((const void*)tmem_slot)), "r"(C::TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = *tmem_slot;

  if (warp < 4) {
    // ------------------------------------------------------------------ softmax and output: a thread a row, whose 128 scores stay in registers
    const int qi = q0 + warp * 32 + lane;
    const uint32_t tS = tmem_base + ((uint32_t)(warp * 32) << 16), tO = tS + 128u;
    const float* ramp = reinterpret_cast<const float*>(smem_raw + C::RAMP);
    const Score f = score_of(p, h);
    const bool cap = p.cap > 0.f;
    // With neither a cap nor slopes the scale goes into the exponent's multiply-add; a negative one would turn the maximum around.
    const bool folded = !cap && f.slope == 0.f && p.scale > 0.f;
    const float unit = folded ? f.post : 1.f, post = folded ? 1.f : f.post;
    int lo, hi, own = 0;
    row_span(p, qi, prefix, lo, hi);
    if (qi >= p.Tq) hi = -1;
    if (p.seg_q != nullptr) own = qi < p.Tq ? p.seg_q[(long long)b * p.Tq + qi] : -1;
    float m = -INFINITY;  // maximum that P is relative to, in log2
    uint64_t l2[2] = {0, 0};
    const bool short_cap = cap && f.slope == 0.f && c_.folds && p.scale > 0.f;
    bool ok = true;
    int count = 0;  // tiles so far
    for (int n = next(-1); n < end; n = next(n)) {
      const int k0 = (first + n) * BLK;
      const bool whole = (flags[n] & WHOLE) != 0;
      uint32_t keep[4] = {~0u, ~0u, ~0u, ~0u};
      if (!whole) {  // while the score product runs
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          keep[c] = span_bits(lo, hi, k0 + 32 * c);
          if (p.seg_k != nullptr) {
            const int k = k0 + 32 * c + lane;
            keep[c] &= segment_bits(k < p.Tk ? p.seg_k[(long long)b * p.Tk + k] : -1, own);
          }
        }
      }
      ok = __all_sync(0xffffffffu, mbar_wait(s_full, count & 1, abort_flag));
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const bool plain = folded && whole;
      bool poly = short_cap && whole;
      float x[4][32], m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, offset = 0.f, top = 0.f;
      tmem_ld32(tS, reinterpret_cast<uint32_t*>(x[0]));
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        loaded(x[c]);
        if (c < 3) tmem_ld32(tS + 32u * (c + 1), reinterpret_cast<uint32_t*>(x[c + 1]));
        extremes(x[c], m4, top, plain || poly, poly);
      }
      if (poly && __any_sync(0xffffffffu, top * fabsf(c_.pre) > 0.75f)) {
        poly = false;
        m4[0] = m4[1] = m4[2] = m4[3] = -INFINITY;
      }
      if (!plain && !poly) offset = finish_scores(x, tS, m4, cap, c_, post, f.slope, qi - k0, ramp, whole, keep, __all_sync(0xffffffffu, qi - k0 >= BLK - 1));
      float mx = max_nan(max_nan(m4[0], m4[1]), max_nan(m4[2], m4[3]));
      if (mx != -INFINITY) mx = poly ? tanh_small(mx * c_.pre) * c_.post : folded ? mx * f.post : mx + offset;
      const float m_new = max_nan(m, mx);
      // a NaN or +inf among the scores makes the row NaN, whichever way its exponential goes
      l2[0] = add_f32x2(l2[0], pack_f32x2(m_new == -INFINITY ? 0.f : m_new - m_new, 0.f));
      const bool grow = m_new > m + RESCALE || (m == -INFINITY && m_new > m);
      if (__any_sync(0xffffffffu, grow)) {
        const float alpha = grow ? ex2(m - m_new) : 1.f;
        if (grow) m = m_new;
        const uint64_t a2 = both(alpha);
        l2[0] = mul_f32x2(l2[0], a2);
        l2[1] = mul_f32x2(l2[1], a2);
        if (count > 0) {  // a full S also says that P V of the tile before has been added
#pragma unroll 1
          for (int c = 0; c < D / 16; ++c) {
            uint32_t o[16];
            tmem_ld16(tO + (uint32_t)(c * 16), o);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tmem_st16(tO + (uint32_t)(c * 16), o);
          }
        }
      }
      const uint64_t minus2 = both(m == -INFINITY ? 0.f : offset - m), scale2 = both(unit);
      const uint64_t b0 = both(c_.mid_raw[0]), b1 = both(c_.mid_raw[1]), b2 = both(c_.mid_raw[2]), b3 = both(c_.mid_raw[3]), b4 = both(c_.mid_raw[4]);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if (poly)  // tanh's last product and the subtraction of the maximum are one multiply-add
          exponentials<T, TRAIN>(x[c], tS + (uint32_t)(c * 16), l2, [&](uint64_t v) {
            const uint64_t u = mul_f32x2(v, v);
            return fma_f32x2(fma_f32x2(fma_f32x2(fma_f32x2(fma_f32x2(b4, u, b3), u, b2), u, b1), u, b0), v, minus2);
          });
        else
          exponentials<T, TRAIN>(x[c], tS + (uint32_t)(c * 16), l2, [&](uint64_t v) { return fma_f32x2(v, scale2, minus2); });
        if (c >= 2) {  // the product with the values begins with three quarters of them
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
          __syncwarp();
          if (lane == 0) mbar_arrive(p_ready(c - 2));
        }
      }
      ++count;
    }
    if (ok && count > 0) {
      ok = __all_sync(0xffffffffu, mbar_wait(o_done, 0, abort_flag));
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    }
    if (ok) {
      float la, lb, lc, ld;
      unpack_f32x2(l2[0], la, lb);
      unpack_f32x2(l2[1], lc, ld);
      const float l = (la + lb) + (lc + ld);
      const bool blank = (m == -INFINITY && l == l) || qi >= p.Tq;
      const float inv = blank ? 0.f : 1.f / l;
      // the row, and what its rounding lost
      const long long at = (((long long)b * p.Tq + min(qi, p.Tq - 1)) * p.H + h) * p.D;
#pragma unroll 1
      for (int col = 0; col < D; col += 32) {
        float x[32];
        if (count > 0) {
          tmem_ld32(tO + (uint32_t)col, reinterpret_cast<uint32_t*>(x));
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          uint32_t w[4], lost[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float v0 = blank ? 0.f : x[u * 8 + 2 * e] * inv, v1 = blank ? 0.f : x[u * 8 + 2 * e + 1] * inv;
            float r0, r1;
            w[e] = pack_16<T>(v0, v1);
            unpack_16<T>(w[e], r0, r1);
            lost[e] = pack_16<T>(v0 - r0, v1 - r1);
          }
          if (qi < p.Tq && col + u * 8 < p.D) {
            *reinterpret_cast<uint4*>(o + at + col + u * 8) = make_uint4(w[0], w[1], w[2], w[3]);
            if (TRAIN) *reinterpret_cast<uint4*>(lo_out + at + col + u * 8) = make_uint4(lost[0], lost[1], lost[2], lost[3]);
          }
        }
      }
      if (TRAIN && qi < pitch) lse[((long long)b * p.H + h) * pitch + qi] = blank ? INFINITY : m + log2f(l);
    }
    if (!ok) {
      if (lane == 0 && err) atomicExch(err, 43);
      *abort_flag = 1;
    }
  } else {
    const int start = next(-1);
    if (warp == 4) {
      // ------------------------------------------------------------------ TMA producer
      if (elect_one() && start < end) {
        mbar_expect_tx(q_bar, TILE);
#pragma unroll
        for (int c = 0; c < C::CH; ++c) tma_load_4d(sQ + c * 16384, &map_q, q_bar, c * 64, q0, h, b);  // rows beyond the last query arrive as zeros
        bool ok = true;
        int issued = 0;
        for (int n = start; n < end && ok; n = next(n)) {
          const int k0 = (first + n) * BLK;
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            const int s = issued % RING;
            ok = mbar_wait(kv_empty(s), ((issued / RING) & 1) ^ 1, abort_flag);
            if (!ok) break;
            mbar_expect_tx(kv_full(s), TILE);
            const uint32_t dst = sKV + s * TILE;
            if (kv == 0) {
#pragma unroll
              for (int c = 0; c < C::CH; ++c) tma_load_4d(dst + c * 16384, &map_k, kv_full(s), c * 64, k0, hkv, b);
            } else {
#pragma unroll
              for (int c = 0; c < C::CH; ++c) tma_load_4d(dst + c * 16384, &map_v, kv_full(s), c * 64, k0, hkv, b);
            }
            ++issued;
          }
        }
        if (!ok) {
          if (err) atomicExch(err, 41);
          *abort_flag = 1;
          for (uint32_t spin = 0; spin < (1u << 16); ++spin)
            if (mbar_try_wait(q_bar, 0)) break;
          for (int n = max(0, issued - RING); n < issued; ++n)
            for (uint32_t spin = 0; spin < (1u << 16); ++spin)
              if (mbar_try_wait(kv_full(n % RING), (n / RING) & 1)) break;
        }
      }
    } else {
      // ------------------------------------------------------------------ MMA issuer: the whole warp walks, one lane issues
      const bool leader = elect_one();
      if (start < end) {
        constexpr uint32_t idesc_s = product_desc<T>(128, 128, false), idesc_o = product_desc<T>(128, D, true);
        const uint64_t q_desc = make_smem_desc(sQ, false), k_desc = make_smem_desc(sKV, false), v_desc = mn_desc(sKV, 16384);
        const uint32_t tO = tmem_base + 128u;
        auto scores = [&](int s) {
          const uint64_t bd = k_desc + (uint64_t)((uint32_t)(s * TILE) >> 4);
          if (leader) {
#pragma unroll
            for (int c = 0; c < C::CH; ++c)
#pragma unroll
              for (int k = 0; k < 4; ++k) umma_bf16(tmem_base, q_desc + (uint64_t)(c * 1024 + 2 * k), bd + (uint64_t)(c * 1024 + 2 * k), idesc_s, (c > 0 || k > 0) ? 1u : 0u);
            umma_commit(s_full);
            umma_commit(kv_empty(s));
          }
        };
        auto values = [&](int s, int from, int to, bool fresh) {
          const uint64_t bd = v_desc + (uint64_t)((uint32_t)(s * TILE) >> 4);
          if (leader) {
#pragma unroll
            for (int k = 0; k < 8; ++k)  // 16 keys: 8 columns of packed pairs
              if (k >= from && k < to) {
                umma_bf16_ts(tO, tmem_base + (uint32_t)(k * 8), bd + (uint64_t)((2048u >> 4) * k), idesc_o, (!fresh || k > 0) ? 1u : 0u);
                if (TRAIN) umma_bf16_ts(tO, tmem_base + (uint32_t)(64 + k * 8), bd + (uint64_t)((2048u >> 4) * k), idesc_o, 1u);
              }
          }
        };
        auto wait = [&](uint32_t bar, int nth) {
          const bool there = __all_sync(0xffffffffu, mbar_wait(bar, nth & 1, abort_flag));
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          return there;
        };
        int done = 0, at = 0;  // tiles so far; ring position of K(n); V(n) follows it, then K of the next tile
        bool ok = wait(q_bar, 0) && wait(kv_full(0), 0);
        if (ok) scores(0);
        for (int n = start; n < end && ok; at += 2, ++done) {
          const int then = next(n), sv = (at + 1) % RING, sk = (at + 2) % RING;
          ok = wait(kv_full(sv), (at + 1) / RING) && (then >= end || wait(kv_full(sk), (at + 2) / RING)) && wait(p_ready(0), done);
          if (!ok) break;
          values(sv, 0, 6, done == 0);  // P is in TMEM, S has been read, O rescaled
          ok = wait(p_ready(1), done);
          if (!ok) break;
          values(sv, 6, 8, false);
          if (leader) umma_commit(kv_empty(sv));
          if (then < end) scores(sk);
          else if (leader) umma_commit(o_done);
          n = then;
        }
        if (!ok) {
          if (leader && err) atomicExch(err, 42);
          *abort_flag = 1;
        }
      }
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  __syncwarp();
  if (warp == 5) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(C::TMEM_COLS) : "memory");
  }
}

template <typename T, int D, bool TRAIN>
int launch_fwd(const CUtensorMap* maps, const Rules& p, void* o, void* lo, float* lse, int pitch, int* err, cudaStream_t stream) {
  using C = FwdCfg<D>;
  const int smem = C::SMEM + ((p.Tk + BLK - 1) / BLK + 15) / 16 * 16;
  static bool attr[KB_MAX_DEVICES] = {false};
  if (!kb_allow_smem(rules_fwd_sm100<T, D, TRAIN>, C::SMEM + MAX_BLOCKS, attr)) {
    kb200_set_error("attention_rules: shared-memory limit");
    return -3;
  }
  const long long grid = (long long)((p.Tq + BLK - 1) / BLK) * p.H * p.B;
  rules_fwd_sm100<T, D, TRAIN><<<(unsigned)grid, C::THREADS_, smem, stream>>>(maps[0], maps[1], maps[2], p, make_cap(p.scale, p.cap), (T*)o, (T*)lo, lse, pitch, err);
  return 0;
}

}  // namespace

// As kb200_attention_rules_fwd for 16-bit types (dtype 1 bfloat16, 2 float16) and D a multiple of 8 up to 128, base pointers and strides multiples of
// 16 bytes, at most 1048576 keys.  lo (null with lse): [B, Tq, H, D], what rounding o lost.  lse rows are `pitch` apart; those beyond Tq get +inf.
KB_API int kb200_attention_rules_fwd_sm100(const void* q, const void* k, const void* v, void* o, void* lo, float* lse, int pitch, const long long* strides, int dtype, int B, int H,
                                           int Hkv, int Tq, int Tk, int D, int* err, float scale, float cap, const float* slopes, int causal, int window, const int* prefix,
                                           const int* seg_q, const int* seg_k, const void* range_q, const void* range_k, cudaStream_t stream) {
  const Rules p{B, H, Hkv, Tq, Tk, D, scale, cap, slopes, causal, window, prefix, seg_q, seg_k, (const int4*)range_q, (const int4*)range_k};
  if (B <= 0 || H <= 0 || Hkv <= 0 || H % Hkv || Tq <= 0 || Tk <= 0 || D <= 0 || D > 128 || D % 8 || (dtype != 1 && dtype != 2) || Tk > MAX_BLOCKS * BLK ||
      (long long)((Tq + 127) / 128) * H * B > 0x7fffffffll) {
    kb200_set_error("attention_rules_fwd_sm100: sizes out of range");
    return -2;
  }
  const Strides qs{strides[0], strides[1], strides[2]}, ks{strides[3], strides[4], strides[5]}, vs{strides[6], strides[7], strides[8]};
  if (!rules_strides(qs, q, Tq, H, B) || !rules_strides(ks, k, Tk, Hkv, B) || !rules_strides(vs, v, Tk, Hkv, B) || (((uintptr_t)o | (uintptr_t)lo) & 15)) {
    kb200_set_error("attention_rules_fwd_sm100: strides and base pointers must be multiples of 16 bytes");
    return -2;
  }
  if ((lo == nullptr) != (lse == nullptr) || (lse != nullptr && pitch < Tq)) {
    kb200_set_error("attention_rules_fwd_sm100: lo and lse go together");
    return -2;
  }
  const bool half = dtype == 2;
  CUtensorMap maps[3];
  if (!rules_map(&maps[0], q, D, Tq, H, B, qs, 128, half) || !rules_map(&maps[1], k, D, Tk, Hkv, B, ks, 128, half) || !rules_map(&maps[2], v, D, Tk, Hkv, B, vs, 128, half)) {
    kb200_set_error("attention_rules_fwd_sm100: cuTensorMapEncodeTiled failed");
    return -3;
  }
  int rc;
#define KB_TRAIN(T, DD) (lse != nullptr ? launch_fwd<T, DD, true>(maps, p, o, lo, lse, pitch, err, stream) : launch_fwd<T, DD, false>(maps, p, o, lo, lse, pitch, err, stream))
#define KB_CALL(DD) (half ? KB_TRAIN(__half, DD) : KB_TRAIN(__nv_bfloat16, DD))
  rc = D <= 64 ? KB_CALL(64) : KB_CALL(128);
#undef KB_CALL
#undef KB_TRAIN
  if (rc != 0) return rc;
  KB_CHECK_LAUNCH("attention_rules_fwd_sm100");
  return 0;
}
