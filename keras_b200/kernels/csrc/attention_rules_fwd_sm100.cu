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
  static constexpr int FLAGS = BARS + 256;
  static constexpr int SMEM = FLAGS;  // and a byte a tile of keys
  static constexpr uint32_t TMEM_COLS = NT == 2 ? 512 : 256;
  static constexpr int THREADS_ = NT == 2 ? 384 : 192;
};
constexpr float RESCALE = 8.f;

template <typename T, int D, int NT>
__global__ void __launch_bounds__(FwdCfg<D, NT>::THREADS_, NT == 2 ? 1 : 2)
rules_fwd_sm100(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                const __grid_constant__ CUtensorMap map_o, const __grid_constant__ CUtensorMap map_lo, const Rules p, float* lse, int pitch, int with_lo, int* err) {
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
  auto p_ready = [&](int n) { return bar_base + 8u * (1 + 2 * RING + NT + n); };  // tile i: 2i its first 64 keys, 2i + 1 the rest
  auto o_done = [&](int i) { return bar_base + 8u * (1 + 2 * RING + 3 * NT + i); };
  constexpr int N_BARS = 1 + 2 * RING + 4 * NT;
  static_assert(N_BARS * 8 + 8 <= 256, "barrier area");
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
      mbar_init(p_ready(2 * i), 4);
      mbar_init(p_ready(2 * i + 1), 4);
      mbar_init(o_done(i), 1);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 4 * NT + 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32((const void*)tmem_slot)), "r"(C::TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = *tmem_slot;
  const int end = last - first + 1;

  // NT = 2: 384 threads x 168 registers at launch = 256 x 224 + 128 x 56
  if (warp < 4 * NT) {
    if constexpr (NT == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    // ------------------------------------------------------------------ softmax and output, one thread per query row
    const int i = warp >> 2, q = warp & 3;
    const int row = q * 32 + lane, qi = q0 + i * BLK + row;
    const uint32_t lane_base = (uint32_t)(q * 32) << 16;
    const uint32_t tS = tmem_base + (uint32_t)(i * 128) + lane_base, tO = tmem_base + (uint32_t)(NT * 128 + i * D) + lane_base;
    const Score f = score_of(p, h);
    const bool cap = p.cap > 0.f;
    // with neither a cap nor slopes the scale goes into the exponent's multiply-add
    const bool folded = !cap && f.slope == 0.f && f.post > 0.f;
    const float unit = folded ? f.post : 1.f;
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
      const int k0 = (first + n) * BLK;
      uint32_t keep[4] = {~0u, ~0u, ~0u, ~0u};
      if (!(fl & WHOLE)) {  // this row's 128 bits, while the score product runs
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          keep[c] = span_bits(lo, hi, k0 + c * 32);
          if (p.seg_k != nullptr) {
            const int k = k0 + c * 32 + lane;
            keep[c] &= segment_bits(k < p.Tk ? p.seg_k[(long long)b * p.Tk + k] : -1, own);
          }
        }
      }
      ok = mbar_wait(s_full(i), count & 1, abort_flag);
      if (!(ok = __all_sync(0xffffffffu, ok))) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      float x[128];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32(tS + (uint32_t)(c * 32), reinterpret_cast<uint32_t*>(x) + c * 32);
      asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
      if (cap) {
        capped(x, f.pre);
        const uint64_t post2 = both(f.post);
#pragma unroll
        for (int e = 0; e < 128; e += 2) unpack_f32x2(mul_f32x2(pack_f32x2(x[e], x[e + 1]), post2), x[e], x[e + 1]);
      } else if (!folded) {
#pragma unroll
        for (int e = 0; e < 128; ++e) x[e] *= f.post;
      }
      if (f.slope != 0.f) {
        const float from = (float)(qi - k0);
#pragma unroll
        for (int e = 0; e < 128; ++e) x[e] = fmaf(-f.slope, fabsf(from - (float)e), x[e]);
      }
      if (!(fl & WHOLE)) {
#pragma unroll
        for (int e = 0; e < 128; ++e)
          if (!(keep[e >> 5] >> (e & 31) & 1u)) x[e] = -INFINITY;
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int e = 0; e < 128; e += 8)
#pragma unroll
        for (int c = 0; c < 4; ++c) mx[c] = max_nan(mx[c], max_nan(x[e + c], x[e + 4 + c]));
      const float m_new = max_nan(m, max_nan(max_nan(mx[0], mx[1]), max_nan(mx[2], mx[3])) * unit);
      // a NaN or +inf among the scores makes the row NaN, whichever way its exponential goes
      l2[0] = add_f32x2(l2[0], pack_f32x2(m_new == -INFINITY ? 0.f : m_new - m_new, 0.f));
      const bool grow = m_new > m + RESCALE || (m == -INFINITY && m_new > m);
      if (__any_sync(0xffffffffu, grow)) {
        const float alpha = grow ? ex2(m - m_new) : 1.f;
        if (grow) m = m_new;
        const uint64_t a2 = both(alpha);
        l2[0] = fma_f32x2(l2[0], a2, 0);
        l2[1] = fma_f32x2(l2[1], a2, 0);
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
      const uint64_t scale2 = both(unit), minus2 = both(m == -INFINITY ? 0.f : -m);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float x0, x1;
          const uint64_t x2 = fma_f32x2(pack_f32x2(x[c * 32 + 2 * e], x[c * 32 + 2 * e + 1]), scale2, minus2);
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
        if (c & 1) {  // 64 keys are there: P V may start on them
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
          __syncwarp();
          if (lane == 0) mbar_arrive(p_ready(2 * i + (c >> 1)));
        }
      }
      ++count;
    }
    if (ok && count > 0) {
      ok = __all_sync(0xffffffffu, mbar_wait(o_done(i), 0, abort_flag));
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    } else if (ok && next(-1) < end) {
      ok = __all_sync(0xffffffffu, mbar_wait(q_bar, 0, abort_flag));  // zeros are staged where Q may still be on its way, for the other tile's sake
    }
    if (ok) {
      float la, lb, lc, ld;
      unpack_f32x2(l2[0], la, lb);
      unpack_f32x2(l2[1], lc, ld);
      const float l = (la + lb) + (lc + ld);
      const bool blank = (m == -INFINITY && l == l) || qi >= p.Tq;
      const float inv_l = blank ? 0.f : 1.f / l;
      // every product of this tile has completed: its Q is free, O is staged there; then what O's rounding lost, where it is asked for
#pragma unroll 1
      for (int part = 0; part <= with_lo; ++part) {
        if (part > 0) {
          if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
          __syncwarp();
        }
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          float o[32];
          if (count > 0) {
            tmem_ld32(tO + (uint32_t)(c * 32), reinterpret_cast<uint32_t*>(o));
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
          }
          const uint32_t chunk = sQ + (uint32_t)(i * TILE + (c >> 1) * 16384) + (uint32_t)row * 128u;
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float v0 = blank ? 0.f : o[u * 8 + 2 * e] * inv_l, v1 = blank ? 0.f : o[u * 8 + 2 * e + 1] * inv_l;
              w[e] = pack_16<T>(v0, v1);
              if (part > 0) {
                float r0, r1;
                unpack_16<T>(w[e], r0, r1);
                w[e] = pack_16<T>(v0 - r0, v1 - r1);
              }
            }
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(chunk + (((uint32_t)((c & 1) * 4 + u) ^ (uint32_t)(row & 7)) << 4)), "r"(w[0]), "r"(w[1]),
                         "r"(w[2]), "r"(w[3]) : "memory");
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0 && q0 + i * BLK + q * 32 < p.Tq) {
#pragma unroll
          for (int c = 0; c < D / 64; ++c)
            tma_store_4d(part == 0 ? &map_o : &map_lo, sQ + (uint32_t)(i * TILE + c * 16384) + (uint32_t)(q * 32) * 128u, c * 64, q0 + i * BLK + q * 32, h, b);
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
      }
      if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");  // the writes land before the grid ends
      if (lse != nullptr && qi < pitch) lse[((long long)b * p.H + h) * pitch + qi] = blank ? INFINITY : m + log2f(l);
    }
    if (!ok) {
      if (lane == 0 && err) atomicExch(err, 43);
      *abort_flag = 1;
    }
  } else {
    if constexpr (NT == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    const int start = next(-1);
    if (warp == 4 * NT) {
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
    } else if (warp == 4 * NT + 1) {
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
        auto values = [&](int i, int s, int half, bool fresh) {  // 64 keys
          const uint64_t bdesc = mn_desc(sKV + s * TILE + half * 8192, 16384);
#pragma unroll
          for (int k = 0; k < 4; ++k)  // 16 keys: 8 columns of packed pairs
            umma_bf16_ts(tmem_O(i), tmem_S(i) + (uint32_t)(half * 32 + k * 8), bdesc + (uint64_t)((2048u >> 4) * k), idesc_o, (!fresh || half > 0 || k > 0) ? 1u : 0u);
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
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                if (ok) ok = mbar_wait(p_ready(2 * i + half), done[i] & 1, abort_flag);  // that half of P is in TMEM, S has been read, O rescaled
                if (!ok) continue;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                values(i, nv % RING, half, done[i] == 0);
              }
              if (!ok) continue;
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
  if (warp == 4 * NT + 1) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(C::TMEM_COLS) : "memory");
  }
}

template <typename T, int D, int NT>
int launch_fwd(const CUtensorMap* maps, const Rules& p, float* lse, int pitch, int with_lo, int* err, cudaStream_t stream) {
  using C = FwdCfg<D, NT>;
  const int smem = C::SMEM + ((p.Tk + BLK - 1) / BLK + 15) / 16 * 16;
  static bool attr[KB_MAX_DEVICES] = {false};
  if (!kb_allow_smem(rules_fwd_sm100<T, D, NT>, C::SMEM + MAX_BLOCKS, attr)) {
    kb200_set_error("attention_rules: shared-memory limit");
    return -3;
  }
  const long long grid = (long long)((p.Tq + 128 * NT - 1) / (128 * NT)) * p.H * p.B;
  rules_fwd_sm100<T, D, NT><<<(unsigned)grid, C::THREADS_, smem, stream>>>(maps[0], maps[1], maps[2], maps[3], maps[4], p, lse, pitch, with_lo, err);
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
  const Strides os{(long long)H * D, D, (long long)Tq * H * D};
  if (!rules_strides(qs, q, Tq, H, B) || !rules_strides(ks, k, Tk, Hkv, B) || !rules_strides(vs, v, Tk, Hkv, B) || (((uintptr_t)o | (uintptr_t)lo) & 15)) {
    kb200_set_error("attention_rules_fwd_sm100: strides and base pointers must be multiples of 16 bytes");
    return -2;
  }
  const bool half = dtype == 2;
  CUtensorMap maps[5];
  if (!rules_map(&maps[0], q, D, Tq, H, B, qs, 128, half) || !rules_map(&maps[1], k, D, Tk, Hkv, B, ks, 128, half) || !rules_map(&maps[2], v, D, Tk, Hkv, B, vs, 128, half) ||
      !rules_map(&maps[3], o, D, Tq, H, B, os, 32, half) || !rules_map(&maps[4], lo != nullptr ? lo : o, D, Tq, H, B, os, 32, half)) {
    kb200_set_error("attention_rules_fwd_sm100: cuTensorMapEncodeTiled failed");
    return -3;
  }
  const int with_lo = lo != nullptr ? 1 : 0;
  int rc;
#define KB_CALL(DD, NT) (half ? launch_fwd<__half, DD, NT>(maps, p, lse, pitch, with_lo, err, stream) : launch_fwd<__nv_bfloat16, DD, NT>(maps, p, lse, pitch, with_lo, err, stream))
  if (D <= 64) rc = Tq <= 128 ? KB_CALL(64, 1) : KB_CALL(64, 2);
  else rc = Tq <= 128 ? KB_CALL(128, 1) : KB_CALL(128, 2);
#undef KB_CALL
  if (rc != 0) return rc;
  KB_CHECK_LAUNCH("attention_rules_fwd_sm100");
  return 0;
}
