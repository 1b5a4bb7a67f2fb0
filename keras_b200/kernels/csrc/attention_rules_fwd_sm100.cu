// Attention with scores by rule, forward pass on tcgen05 tensor cores, for 16-bit heads of up to 128 (multiples of 8; narrower ones are filled
// with zeros by the tile copies).  Same roles as the plain kernel of attention.cu: one thread a row for the softmax, a TMA warp, an MMA warp,
// two tiles of 128 rows a CTA (one for at most 128 rows), P handed over through TMEM, O in TMEM, rescaled only when the maximum grows by
// more than 2^8.
//
// What the rules add:
//   tiles       the flags of every tile of 128 keys (left out / looked at / whole) are worked out once, before the roles part; all of
//               them walk over the same list.  Documents, windows and prefixes cost what they leave visible.
//   cap         tanh as a polynomial on the FMA pipe (packed pairs, 4.5 issue slots a score) while no score of the warp is beyond the cap;
//               the exponentials then stay on the special-function pipe
//   distance    two more instructions a score, in kernels that have slopes
//   masks       32 bits a chunk, in tiles that are not whole; segments by comparing with ids that the warp loads once
// A row that sees nothing keeps a maximum of -inf and becomes zero.
//
// For training the CTA stores L = max + log2(sum) of each row, and beside O the part of it that its rounding lost (`lo`, in 16 bits again):
// the gradient needs sum_d dO O to more than O's own eight bits, or its error would be half as large again.
#include "attention_rules_sm100.cuh"

namespace {
using namespace kbrules;

template <int D, int NT>
struct FwdCfg {
  static constexpr int CH = D / 64;
  static constexpr int TILE = CH * 16384;
  static constexpr int RING = NT == 2 ? (D == 128 ? 4 : 8) : (D == 128 ? 2 : 4);
  static constexpr int BARS = (NT + RING) * TILE;
  static constexpr int FLAGS = BARS + 384 + 2 * NT * 2 * 128 * 4;
  static constexpr int SMEM = FLAGS;  // and a byte a tile of keys
  static constexpr uint32_t TMEM_COLS = NT == 2 ? 512 : 256;
  static constexpr int SOFTMAX = 8 * NT;                 // warps: two threads a row
  static constexpr int THREADS_ = (SOFTMAX + 2) * 32;
  static constexpr int EXCHANGE = BARS + 384;            // [parity][tile][half][row] maxima
};
constexpr float RESCALE = 8.f;

template <typename T, int D, int NT>
__global__ void __launch_bounds__(FwdCfg<D, NT>::THREADS_, NT == 2 ? 1 : 2)
rules_fwd_sm100(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                const Rules p, const Cap c_, T* o, T* lo_out, float* lse, int pitch, int* err) {
  using C = FwdCfg<D, NT>;
  constexpr int TILE = C::TILE, RING = C::RING;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t base = smem_u32(smem_raw);
  if (base & 1023u) {
    if (threadIdx.x == 0 && err) atomicExch(err, 40);
    return;
  }
  const uint32_t sQ = base, sKV = sQ + NT * TILE, bar_base = base + C::BARS;
  uint8_t* flags = smem_raw + C::FLAGS;  // of key tile first + n: two bits each of row tiles 0 and 1
  const uint32_t q_bar = bar_base;
  auto kv_full = [&](int s) { return bar_base + 8u * (1 + s); };
  auto kv_empty = [&](int s) { return bar_base + 8u * (1 + RING + s); };
  auto s_full = [&](int i) { return bar_base + 8u * (1 + 2 * RING + i); };
  auto p_ready = [&](int i) { return bar_base + 8u * (1 + 2 * RING + NT + i); };
  auto o_done = [&](int i) { return bar_base + 8u * (1 + 2 * RING + 2 * NT + i); };
  auto top_ready = [&](int n) { return bar_base + 8u * (1 + 2 * RING + 3 * NT + n); };  // 4 * tile + quarter: both halves of 32 rows have their maximum there
  constexpr int N_BARS = 1 + 2 * RING + 7 * NT;
  static_assert(N_BARS * 8 + 8 <= 384, "barrier area");
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem_raw + C::BARS + N_BARS * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int groups = p.H * p.B, n_q = (p.Tq + 128 * NT - 1) / (128 * NT);
  const int q0 = (n_q - 1 - (int)(blockIdx.x / groups)) * 128 * NT;  // the longest rows of a causal mask first
  const int h = (int)(blockIdx.x % groups) % p.H, b = (int)(blockIdx.x % groups) / p.H;
  const int hkv = h / (p.H / p.Hkv);
  const int prefix = p.prefix != nullptr ? p.prefix[b] : 0;
  int first, last;  // tiles of keys
  keys_of_rows(p, q0, min(q0 + 128 * NT, p.Tq) - 1, prefix, first, last);
  first /= BLK;
  last = last < 0 ? -1 : last / BLK;
  for (int n = threadIdx.x; first + n <= last; n += C::THREADS_) {
    int f = tile_flags(p, b, q0, (first + n) * BLK, prefix);
    if (NT == 2) f |= tile_flags(p, b, q0 + BLK, (first + n) * BLK, prefix) << 2;
    flags[n] = (uint8_t)f;
  }
  auto next = [&](int n) {  // the next tile that any of the rows needs, last - first + 1 if there is none
    do ++n;
    while (first + n <= last && (flags[n] & (NEEDED | NEEDED << 2)) == 0);
    return n;
  };
  auto needs = [&](int i, int n) { return first + n <= last && (flags[n] >> (2 * i) & NEEDED) != 0; };

  if (threadIdx.x == 0) {
    mbar_init(q_bar, 1);
    for (int s = 0; s < RING; ++s) {
      mbar_init(kv_full(s), 1);
      mbar_init(kv_empty(s), 1);
    }
    for (int i = 0; i < NT; ++i) {
      mbar_init(s_full(i), 1);
      mbar_init(p_ready(i), 8);
      mbar_init(o_done(i), 1);
      for (int n = 0; n < 4; ++n) mbar_init(top_ready(4 * i + n), 2);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == C::SOFTMAX + 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32((const void*)tmem_slot)), "r"(C::TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = *tmem_slot;
  const int end = last - first + 1;

  if (warp < C::SOFTMAX) {
    // ------------------------------------------------------------------ softmax and output: two threads a row, each with 64 of its keys
    const int i = warp >> 3, half = warp >> 2 & 1, q = warp & 3;
    const int row = q * 32 + lane, qi = q0 + i * BLK + row;
    const uint32_t lane_base = (uint32_t)(q * 32) << 16;
    const uint32_t tS = tmem_base + (uint32_t)(i * 128 + half * 64) + lane_base, tO = tmem_base + (uint32_t)(NT * 128 + i * D) + lane_base;
    float* exchange = reinterpret_cast<float*>(smem_raw + C::EXCHANGE) + i * 256 + row;
    const Score f = score_of(p, h);
    const bool cap = p.cap > 0.f;
    // Without slopes a row's largest score is that of its largest product, if the scale is positive: the maximum is taken before the scores are
    // made.  With neither a cap nor slopes the scale then goes into the exponent's multiply-add.
    const bool direct = f.slope == 0.f && p.scale > 0.f, folded = direct && !cap;
    const float unit = folded ? f.post : 1.f, post = folded ? 1.f : f.post;
    int lo, hi, own = 0;
    row_span(p, qi, prefix, lo, hi);
    if (qi >= p.Tq) hi = -1;
    if (p.seg_q != nullptr) own = qi < p.Tq ? p.seg_q[(long long)b * p.Tq + qi] : -1;
    float m = -INFINITY;  // maximum that P is relative to, in log2
    uint64_t l2[2] = {0, 0};
    bool ok = true;
    int count = 0;  // tiles so far
    for (int n = next(-1); n < end; n = next(n)) {
      const int fl = flags[n] >> (2 * i);
      if (!(fl & NEEDED)) continue;
      const int k0 = (first + n) * BLK + half * 64;
      const bool whole = (fl & WHOLE) != 0;
      uint32_t keep0 = ~0u, keep1 = ~0u;
      if (!whole) {  // this thread's 64 bits, while the score product runs
        keep0 = span_bits(lo, hi, k0);
        keep1 = span_bits(lo, hi, k0 + 32);
        if (p.seg_k != nullptr) {
          const int k = k0 + lane;
          const int* seg = p.seg_k + (long long)b * p.Tk;
          keep0 &= segment_bits(k < p.Tk ? seg[k] : -1, own);
          keep1 &= segment_bits(k + 32 < p.Tk ? seg[k + 32] : -1, own);
        }
      }
      ok = mbar_wait(s_full(i), count & 1, abort_flag);
      if (!(ok = __all_sync(0xffffffffu, ok))) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      // the maximum; scores are read from TMEM twice, so that only 32 of them are in registers at a time
      float mx = -INFINITY;
#pragma unroll 1
      for (int c = 0; c < 2; ++c) {
        float x[32];
        tmem_ld32(tS + (uint32_t)(c * 32), reinterpret_cast<uint32_t*>(x));
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        if (!direct) scores32(x, cap, c_, post, f.slope, (float)(qi - k0 - c * 32));
        if (!whole) {
          const uint32_t keep = c == 0 ? keep0 : keep1;
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (!(keep >> e & 1u)) x[e] = -INFINITY;
        }
        float m4[4] = {mx, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < 32; e += 8)
#pragma unroll
          for (int u = 0; u < 4; ++u) m4[u] = max3_nan(m4[u], x[e + u], x[e + 4 + u]);
        mx = max_nan(max_nan(m4[0], m4[1]), max_nan(m4[2], m4[3]));
      }
      if (direct && mx != -INFINITY) mx = cap ? tanh_any(mx * f.pre) * f.post : mx * f.post;
      float* slot = exchange + (count & 1) * (NT * 256);
      slot[half * 128] = mx;
      __syncwarp();
      if (lane == 0) mbar_arrive(top_ready(4 * i + q));
      ok = mbar_wait(top_ready(4 * i + q), count & 1, abort_flag);
      if (!(ok = __all_sync(0xffffffffu, ok))) break;
      const float m_new = max3_nan(m, mx, slot[(half ^ 1) * 128]);
      // a NaN or +inf among the scores makes the row NaN, whichever way its exponential goes
      l2[0] = add_f32x2(l2[0], pack_f32x2(m_new == -INFINITY ? 0.f : m_new - m_new, 0.f));
      const bool grow = m_new > m + RESCALE || (m == -INFINITY && m_new > m);
      if (__any_sync(0xffffffffu, grow)) {
        const float alpha = grow ? ex2(m - m_new) : 1.f;
        if (grow) m = m_new;
        const uint64_t a2 = both(alpha);
        l2[0] = fma_f32x2(l2[0], a2, 0);
        l2[1] = fma_f32x2(l2[1], a2, 0);
        if (count > 0) {  // a full S also says that P V of the tile before has been added; each of the two threads takes half of O
#pragma unroll 1
          for (int c = half * (D / 32); c < (half + 1) * (D / 32); ++c) {
            uint32_t o[16];
            tmem_ld16(tO + (uint32_t)(c * 16), o);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tmem_st16(tO + (uint32_t)(c * 16), o);
          }
        }
      }
      const uint64_t scale2 = both(unit), minus2 = both(m == -INFINITY ? 0.f : -m);
#pragma unroll 1
      for (int c = 0; c < 2; ++c) {
        float x[32];
        tmem_ld32(tS + (uint32_t)(c * 32), reinterpret_cast<uint32_t*>(x));
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        scores32(x, cap, c_, post, f.slope, (float)(qi - k0 - c * 32));
        if (!whole) {
          const uint32_t keep = c == 0 ? keep0 : keep1;
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (!(keep >> e & 1u)) x[e] = -INFINITY;
        }
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float x0, x1;
          const uint64_t x2 = fma_f32x2(pack_f32x2(x[2 * e], x[2 * e + 1]), scale2, minus2);
          if (e % 4 == 3 && !cap) {  // a quarter on the FMA pipe, which a cap keeps busy enough
            exp2_poly2(x2, x0, x1);
          } else {
            unpack_f32x2(x2, x0, x1);
            x0 = ex2(x0);
            x1 = ex2(x1);
          }
          l2[e & 1] = add_f32x2(l2[e & 1], pack_f32x2(x0, x1));
          w[e] = pack_16<T>(x0, x1);
        }
        tmem_st16(tS + (uint32_t)(c * 16), w);
      }
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(p_ready(i));
      ++count;
    }
    if (ok && count > 0) {
      ok = __all_sync(0xffffffffu, mbar_wait(o_done(i), 0, abort_flag));
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    }
    if (ok) {
      // both halves add the two sums in one order
      float la, lb, lc, ld;
      unpack_f32x2(l2[0], la, lb);
      unpack_f32x2(l2[1], lc, ld);
      float l = (la + lb) + (lc + ld);
      if (count > 0) {  // the other half's sum: exchanged as the maxima were
        float* slot = exchange + (count & 1) * (NT * 256);
        slot[half * 128] = l;
        __syncwarp();
        if (lane == 0) mbar_arrive(top_ready(4 * i + q));
        ok = __all_sync(0xffffffffu, mbar_wait(top_ready(4 * i + q), count & 1, abort_flag));
        l += slot[(half ^ 1) * 128];
      }
      const bool blank = (m == -INFINITY && l == l) || qi >= p.Tq;
      const float inv_l = blank ? 0.f : 1.f / l;
      // each of the two threads stores half of the row, and what its rounding lost where that is asked for
      const long long at = (((long long)b * p.Tq + min(qi, p.Tq - 1)) * p.H + h) * p.D;
#pragma unroll 1
      for (int col = half * (D / 2); ok && col < (half + 1) * (D / 2); col += 32) {
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
            const float v0 = blank ? 0.f : x[u * 8 + 2 * e] * inv_l, v1 = blank ? 0.f : x[u * 8 + 2 * e + 1] * inv_l;
            float r0, r1;
            w[e] = pack_16<T>(v0, v1);
            unpack_16<T>(w[e], r0, r1);
            lost[e] = pack_16<T>(v0 - r0, v1 - r1);
          }
          if (qi < p.Tq && col + u * 8 < p.D) {
            *reinterpret_cast<uint4*>(o + at + col + u * 8) = make_uint4(w[0], w[1], w[2], w[3]);
            if (lo_out != nullptr) *reinterpret_cast<uint4*>(lo_out + at + col + u * 8) = make_uint4(lost[0], lost[1], lost[2], lost[3]);
          }
        }
      }
      if (lse != nullptr && half == 0 && qi < pitch) lse[((long long)b * p.H + h) * pitch + qi] = blank ? INFINITY : m + log2f(l);
    }
    if (!ok) {
      if (lane == 0 && err) atomicExch(err, 43);
      *abort_flag = 1;
    }
  } else {
    const int start = next(-1);
    if (warp == C::SOFTMAX) {
      // ------------------------------------------------------------------ TMA producer
      if (elect_one() && start < end) {
        mbar_expect_tx(q_bar, NT * TILE);
#pragma unroll
        for (int i = 0; i < NT; ++i)  // rows beyond the last query arrive as zeros
#pragma unroll
          for (int c = 0; c < C::CH; ++c) tma_load_4d(sQ + i * TILE + c * 16384, &map_q, q_bar, c * 64, q0 + i * 128, h, b);
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
      // ------------------------------------------------------------------ MMA issuer
      if (elect_one() && start < end) {
        constexpr uint32_t idesc_s = product_desc<T>(128, 128, false), idesc_o = product_desc<T>(128, D, true);
        auto tmem_S = [&](int i) { return tmem_base + (uint32_t)(i * 128); };
        auto tmem_O = [&](int i) { return tmem_base + (uint32_t)(NT * 128 + i * D); };
        auto scores = [&](int i, int s) {
#pragma unroll
          for (int c = 0; c < C::CH; ++c) {
            const uint64_t adesc = make_smem_desc(sQ + i * TILE + c * 16384, false), bdesc = make_smem_desc(sKV + s * TILE + c * 16384, false);
#pragma unroll
            for (int k = 0; k < 4; ++k) umma_bf16(tmem_S(i), adesc + (uint64_t)(2 * k), bdesc + (uint64_t)(2 * k), idesc_s, (c > 0 || k > 0) ? 1u : 0u);
          }
          umma_commit(s_full(i));
        };
        auto values = [&](int i, int s, bool fresh) {
          const uint64_t bdesc = mn_desc(sKV + s * TILE, 16384);
#pragma unroll
          for (int k = 0; k < 8; ++k)  // 16 keys: 8 columns of packed pairs, those of the second half behind that half's scores
            umma_bf16_ts(tmem_O(i), tmem_S(i) + (uint32_t)((k >> 2) * 64 + (k & 3) * 8), bdesc + (uint64_t)((2048u >> 4) * k), idesc_o, (!fresh || k > 0) ? 1u : 0u);
        };
        int done[NT] = {0}, left[NT] = {0};
        for (int n = start; n < end; n = next(n))
#pragma unroll
          for (int i = 0; i < NT; ++i) left[i] += needs(i, n) ? 1 : 0;
        bool ok = mbar_wait(q_bar, 0, abort_flag) && mbar_wait(kv_full(0), 0, abort_flag);
        if (ok) {
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
          for (int i = 0; i < NT; ++i)
            if (needs(i, start)) scores(i, 0);
          umma_commit(kv_empty(0));
        }
        int at = 0;  // ring position of K(n); V(n) follows it, then K of the next tile
        for (int n = start; n < end && ok; at += 2) {
          const int then = next(n), nv = at + 1, nk = at + 2;
          ok = mbar_wait(kv_full(nv % RING), (nv / RING) & 1, abort_flag);
          if (!ok) break;
          bool have_k = false;
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            if (!ok) continue;
            if (needs(i, n)) {
              ok = mbar_wait(p_ready(i), done[i] & 1, abort_flag);  // P is in TMEM, S has been read, O rescaled
              if (!ok) continue;
              asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
              values(i, nv % RING, done[i] == 0);
              if (++done[i] == left[i]) umma_commit(o_done(i));
            }
            if (needs(i, then)) {
              if (!have_k) ok = mbar_wait(kv_full(nk % RING), (nk / RING) & 1, abort_flag);
              if (!ok) continue;
              have_k = true;
              asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
              scores(i, nk % RING);
            }
          }
          if (!ok) break;
          umma_commit(kv_empty(nv % RING));
          if (then < end) umma_commit(kv_empty(nk % RING));
          n = then;
        }
        if (!ok) {
          if (err) atomicExch(err, 42);
          *abort_flag = 1;
        }
      }
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  __syncwarp();
  if (warp == C::SOFTMAX + 1) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(C::TMEM_COLS) : "memory");
  }
}

template <typename T, int D, int NT>
int launch_fwd(const CUtensorMap* maps, const Rules& p, void* o, void* lo, float* lse, int pitch, int* err, cudaStream_t stream) {
  using C = FwdCfg<D, NT>;
  const int smem = C::SMEM + ((p.Tk + BLK - 1) / BLK + 15) / 16 * 16;
  static bool attr[KB_MAX_DEVICES] = {false};
  if (!kb_allow_smem(rules_fwd_sm100<T, D, NT>, C::SMEM + MAX_BLOCKS, attr)) {
    kb200_set_error("attention_rules: shared-memory limit");
    return -3;
  }
  const long long grid = (long long)((p.Tq + 128 * NT - 1) / (128 * NT)) * p.H * p.B;
  rules_fwd_sm100<T, D, NT><<<(unsigned)grid, C::THREADS_, smem, stream>>>(maps[0], maps[1], maps[2], p, make_cap(p.scale, p.cap), (T*)o, (T*)lo, lse, pitch, err);
  return 0;
}

}  // namespace

// As kb200_attention_rules_fwd for 16-bit types (dtype 1 bfloat16, 2 float16) and D a multiple of 8 up to 128, base pointers and strides multiples of
// 16 bytes, at most 1048576 keys.  lo (may be null): [B, Tq, H, D], what rounding o lost.  lse rows are `pitch` apart; those beyond Tq get +inf.
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
  const bool half = dtype == 2;
  CUtensorMap maps[3];
  if (!rules_map(&maps[0], q, D, Tq, H, B, qs, 128, half) || !rules_map(&maps[1], k, D, Tk, Hkv, B, ks, 128, half) || !rules_map(&maps[2], v, D, Tk, Hkv, B, vs, 128, half)) {
    kb200_set_error("attention_rules_fwd_sm100: cuTensorMapEncodeTiled failed");
    return -3;
  }
  int rc;
#define KB_CALL(DD, NT) (half ? launch_fwd<__half, DD, NT>(maps, p, o, lo, lse, pitch, err, stream) : launch_fwd<__nv_bfloat16, DD, NT>(maps, p, o, lo, lse, pitch, err, stream))
  if (D <= 64) rc = Tq <= 128 ? KB_CALL(64, 1) : KB_CALL(64, 2);
  else rc = Tq <= 128 ? KB_CALL(128, 1) : KB_CALL(128, 2);
#undef KB_CALL
  if (rc != 0) return rc;
  KB_CHECK_LAUNCH("attention_rules_fwd_sm100");
  return 0;
}
