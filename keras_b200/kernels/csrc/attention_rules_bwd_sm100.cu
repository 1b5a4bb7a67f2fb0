// Gradients of attention with scores by rule on tcgen05 tensor cores, for 16-bit heads of up to 128 (attention_rules.cuh says what a score is and
// which keys a row sees; attention_rules.cu has the formulas).  Two kernels without atomics, so that gradients repeat bit for bit:
//
//   rules_dkv  a CTA a tile of 128 keys; walks over the query heads of its group and their tiles of 128 rows.
//              S^T = K Q^T and dP^T = V dO^T in TMEM; P^T and dS^T go back to TMEM in 16 bits, as the operands of dV += P^T dO and dK += dS^T Q
//   rules_dq   a CTA a tile of 128 rows; walks over the tiles of keys.
//              S = Q K^T (two buffers), dP = dO V^T, dS back to TMEM as the operand of dQ += dS K
//
// Sixteen warps work on the scores: four threads a TMEM lane, each with 32 of its 128 columns, so that none needs a shuffle.  With the lane
// a key (dkv) or a row (dq), every operand is a tile as TMA brought it: the same tile is read along its rows for one product and across
// them for the other.  Products run in issue order: S of the next tile may be queued behind the product that reads P from the same columns,
// while the threads are still busy with dS.
// With few key heads a key tile's walk over its query heads is shared out to several CTAs, whose float32 sums a second launch adds up in order
// (6 x 777, 8 query heads on 2, D = 80: dkv 66 -> 44 us).
//
// What bounds them: a tile's chain of product, exponentials, product, gradient, product, of which only the ends overlap with the next tile's: about
// 2300 cycles at D = 128, 3000 with a cap, against 2048 and 1536 of products and 1024 of exponentials.  Both TMEM and shared memory are full, so that
// there is no second CTA to fill the gaps.  Measured at 2 x 4096 x 32/8 x 128: dkv 493 us (1115 TFLOP/s), dq 380 us (1085 TFLOP/s), with a cap 615
// and 465 us; at 8 x 2048 x 16 x 128 with slopes 368 and 269 us; in a window of 1024 at 8192 x 32/8 x 128 with a cap 390 and 284 us.  An issuer that walks as a whole
// warp, and distances without their absolute value, made no difference.
//
// Every mbarrier wait is bounded; on expiry the kernel writes a code to *err, lets its copies land, frees TMEM and returns.
#include <algorithm>

#include "attention_rules_sm100.cuh"

namespace {
using namespace kbrules;

struct Sums {
  const float *lse, *delta;  // [B, H, pitch], pitch a multiple of 128; rows beyond Tq hold +inf and 0
  int pitch;
  const float* peaks;  // float16: [B, H] largest squared norm of a row of dO, then [B, Hkv] of V
};

// dS in float16.  |dS_ij| <= |dP_ij - delta_i| <= 2 max |dO| max |V| (norms of rows; delta is a mean of dP), but with gradients of a mean loss most dS lie far below
// 2^-14, where float16 loses bits and then the value.  So dS goes to its products times the power of two that brings this bound to between 2^14 and 2^15, one of
// a sequence and head (for dK of a key head), and their float32 sums are multiplied with its inverse: exact both ways, as is a gradient that comes
// 2^n times as large or small.  With dO of size 1e-4 at 1 x 4096 x 64 dk was 8.6 times as far off as its own rounding without it, 1.2 times with it.
// bfloat16 has float32's range and needs none.
// Exponent of that power for squares of the norms: 2^x * 2 sqrt(g2 v2) <= 2^15; none where a gradient or the values are zero.
__device__ __forceinline__ int room_of(float g2, float v2) {
  const float square = g2 * v2;  // 7e-15 .. 6e11 each where they are not zero
  return square > 0.f ? 14 - ((((__float_as_int(square) >> 23) & 255) - 127 + 2) >> 1) : 0;
}
__device__ __forceinline__ float power_of_two(int x) { return __int_as_float((x + 127) << 23); }

// Largest squared norm of a row, a block a part of the rows of one sequence and head; rows that are not finite have no say (what they reach is
// NaN whatever the factor).  First the blocks of x, then those of y.  A maximum does not depend on the order of its atomics.  Bound by the bytes of both:
// 8 x 2048 x 16 x 128 23 us (5.9 TB/s), of 790 that the backward pass takes; 6 x 777 x 8/2 x 80 5 us and its clearing 1.
constexpr int PEAK_ROWS = 256;
template <int G>
__global__ void __launch_bounds__(256) peaks_kernel(const __half* x, Strides xs, int T, int H, const __half* y, Strides ys, int Ty, int Hy, float* peaks, int B, int D) {
  const int parts = (T + PEAK_ROWS - 1) / PEAK_ROWS;
  const long long first = (long long)B * H * parts;
  long long at = blockIdx.x;
  int each = parts, heads = H;
  if (at >= first) {
    at -= first;
    peaks += (long long)B * H;
    x = y;
    xs = ys;
    T = Ty;
    heads = Hy;
    each = (Ty + PEAK_ROWS - 1) / PEAK_ROWS;
  }
  const long long unit = at / each;
  const int t0 = (int)(at % each) * PEAK_ROWS, h = (int)(unit % heads), d = (int)(threadIdx.x % G) * 8;
  const __half* from = x + unit / heads * xs.b + h * xs.h + d;
  float top = 0.f;
#pragma unroll 4
  for (int r = threadIdx.x / G; r < PEAK_ROWS; r += 256 / G) {
    uint4 w = make_uint4(0, 0, 0, 0);
    if (t0 + r < T && d < D) w = *reinterpret_cast<const uint4*>(from + (long long)(t0 + r) * xs.t);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float v = __half2float(reinterpret_cast<const __half*>(&w)[i]);
      sum = fmaf(v, v, sum);
    }
#pragma unroll
    for (int n = 1; n < G; n <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, n);
    if (sum <= 3e38f) top = fmaxf(top, sum);
  }
  top = warp_max(top);
  if ((threadIdx.x & 31) == 0 && top > 0.f) atomicMax(reinterpret_cast<int*>(peaks) + unit, __float_as_int(top));  // of floats without a sign, as whole numbers
}
void launch_peaks(const __half* g, const Strides& gs, const __half* v, const Strides& vs, float* peaks, const Rules& p, cudaStream_t stream) {
  cudaMemsetAsync(peaks, 0, (size_t)p.B * (p.H + p.Hkv) * sizeof(float), stream);
  const long long blocks = (long long)p.B * (p.H * (long long)((p.Tq + PEAK_ROWS - 1) / PEAK_ROWS) + p.Hkv * (long long)((p.Tk + PEAK_ROWS - 1) / PEAK_ROWS));
  if (p.D <= 64) peaks_kernel<8><<<(unsigned)blocks, 256, 0, stream>>>(g, gs, p.Tq, p.H, v, vs, p.Tk, p.Hkv, peaks, p.B, p.D);
  else peaks_kernel<16><<<(unsigned)blocks, 256, 0, stream>>>(g, gs, p.Tq, p.H, v, vs, p.Tk, p.Hkv, peaks, p.B, p.D);
}

// From 32 raw scores (columns e of a lane) to probabilities x and w = P (1 - tanh^2).  `from` - e is the distance of the pair; minus_lse(e): of
// columns e and e + 1.
template <typename Lse>
__device__ __forceinline__ void probabilities(float (&x)[32], float (&w)[32], const Score& f, bool cap, const Cap& c, float from, uint32_t keep, bool whole, Lse minus_lse) {
  const bool folded = !cap && f.slope == 0.f;
  scores32(x, cap, c, folded ? 1.f : f.post, f.slope, from);
  if (cap) {
    const uint64_t inv2 = both(-c.inv_post * c.inv_post);
    if (f.slope == 0.f) {
#pragma unroll
      for (int e = 0; e < 32; e += 2) {
        const uint64_t t = pack_f32x2(x[e], x[e + 1]);
        unpack_f32x2(fma_f32x2(mul_f32x2(t, inv2), t, both(1.f)), w[e], w[e + 1]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 32; ++e) {  // the score without its distance
        const float t = fmaf(f.slope, fabsf(from - (float)e), x[e]) * c.inv_post;
        w[e] = fmaf(-t, t, 1.f);
      }
    }
  }
  const uint64_t scale2 = both(folded ? f.post : 1.f);
#pragma unroll
  for (int e = 0; e < 32; e += 2) unpack_f32x2(fma_f32x2(pack_f32x2(x[e], x[e + 1]), scale2, minus_lse(e)), x[e], x[e + 1]);
  if (!whole) {
#pragma unroll
    for (int e = 0; e < 32; ++e)
      if (!(keep >> e & 1u)) x[e] = -INFINITY;
  }
#pragma unroll
  for (int e = 0; e < 32; ++e) {
    x[e] = ex2(x[e]);
    w[e] = cap ? w[e] * x[e] : x[e];
  }
}

// A key tile's walk over the query heads of its group and their row tiles, and the part of it that a CTA takes.
struct Parts {
  int count;    // parts of a key tile; 1: its gradients are stored as they are
  float* sums;  // [dk, dv][count][B, Tk, Hkv, D]
};

// 32 columns of a row in float32 times a power of two, or zeros.
__device__ __forceinline__ void store_sums(float* to, uint32_t tmem, int col, int D, float factor, bool valid, bool zero) {
  float o[32];
  if (!zero) {
    tmem_ld32(tmem, reinterpret_cast<uint32_t*>(o));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
  }
#pragma unroll
  for (int u = 0; u < 8; ++u)
    if (valid && col + u * 4 < D)
      *reinterpret_cast<float4*>(to + col + u * 4) = zero ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(o[u * 4] * factor, o[u * 4 + 1] * factor, o[u * 4 + 2] * factor, o[u * 4 + 3] * factor);
}

// dk and dv from the sums of their parts, in order.
template <typename T>
__global__ void __launch_bounds__(256) join_parts_kernel(const float4* sums, T* dk, T* dv, int parts, long long n, float scale) {
  const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
  if (at >= 2 * n) return;
  const bool second = at >= n;
  const long long e = second ? at - n : at;
  const float4* from = sums + (second ? (long long)parts * n : 0) + e;
  float4 x = from[0];
  for (int i = 1; i < parts; ++i) {
    const float4 y = from[i * n];
    x.x += y.x;
    x.y += y.y;
    x.z += y.z;
    x.w += y.w;
  }
  const float f = second ? 1.f : scale;
  reinterpret_cast<uint2*>(second ? dv : dk)[e] = make_uint2(pack_16<T>(x.x * f, x.y * f), pack_16<T>(x.z * f, x.w * f));
}

// Pulls the tail of a 32-column slice of TMEM into 16-byte stores of one row.
template <typename T>
__device__ __forceinline__ void store_row(T* to, uint32_t tmem, int col, int D, float factor, bool valid, bool zero) {
  float o[32];
  if (!zero) {
    tmem_ld32(tmem, reinterpret_cast<uint32_t*>(o));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = zero ? 0u : pack_16<T>(o[u * 8 + 2 * e] * factor, o[u * 8 + 2 * e + 1] * factor);
    if (valid && col + u * 8 < D) *reinterpret_cast<uint4*>(to + col + u * 8) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

constexpr int BWD_THREADS = 576;  // 16 warps on the scores, one for copies, one for products

// ------------------------------------------------------------------------------------------------ dK, dV
template <int D>
struct DkvCfg {
  static constexpr int CH = D / 64, TILE = CH * 16384, STAGES = D == 128 ? 2 : 4, STAGE = 2 * TILE;
  static constexpr int BARS = 2 * TILE + STAGES * STAGE, SUMS = BARS + 256, FLAGS = SUMS + STAGES * 1024;
};

template <typename T, int D>
__global__ void __launch_bounds__(BWD_THREADS, 1)
rules_dkv_sm100(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                const __grid_constant__ CUtensorMap map_g, const Rules p, const Cap c_, const Sums sums, T* dk, T* dv, const Parts parts, int* err) {
  using C = DkvCfg<D>;
  constexpr int TILE = C::TILE, ST = C::STAGES;
  constexpr bool RANGE = __is_same(T, __half);
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t base = smem_u32(smem_raw);
  if (base & 1023u) {
    if (threadIdx.x == 0 && err) atomicExch(err, 50);
    return;
  }
  const uint32_t sK = base, sV = base + TILE, sQG = base + 2 * TILE, bar_base = base + C::BARS;
  uint8_t* flags = smem_raw + C::FLAGS;
  const uint32_t kv_bar = bar_base, s_full = bar_base + 8, dp_full = bar_base + 16, p_ready = bar_base + 24, ds_ready = bar_base + 32, all_done = bar_base + 40;
  auto full = [&](int s) { return bar_base + 48u + 8u * s; };
  auto empty = [&](int s) { return bar_base + 48u + 8u * (ST + s); };
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem_raw + C::BARS + 48 + 16 * ST);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int unit = (int)(blockIdx.x / parts.count), part = (int)(blockIdx.x % parts.count);
  const int groups = p.Hkv * p.B, k0 = unit / groups * BLK;  // a causal mask gives the first keys the most rows
  const int hkv = unit % groups % p.Hkv, b = unit % groups / p.Hkv, group = p.H / p.Hkv;
  const int prefix = prefix_of(p, b);
  int first, last;  // tiles of rows
  rows_of_keys(p, k0, min(k0 + BLK, p.Tk) - 1, prefix, first, last);
  first /= BLK;
  last = last < 0 ? -1 : last / BLK;
  int* n_needed = reinterpret_cast<int*>(smem_raw + C::BARS + 64 + 16 * ST);
  if (threadIdx.x == 0) *n_needed = 0;
  __syncthreads();
  int needed = 0;
  for (int n = threadIdx.x; first + n <= last; n += BWD_THREADS) {
    const int f = tile_flags(p, b, (first + n) * BLK, k0, prefix);
    flags[n] = (uint8_t)f;
    needed += f & NEEDED;
  }
  if (needed > 0) atomicAdd(n_needed, needed);
  const int end = last - first + 1;
  auto next = [&](int n) {
    do ++n;
    while (n < end && !(flags[n] & NEEDED));
    return n;
  };
  if (threadIdx.x == 0) {
    mbar_init(kv_bar, 1);
    mbar_init(s_full, 1);
    mbar_init(dp_full, 1);
    mbar_init(p_ready, 16);
    mbar_init(ds_ready, 16);
    mbar_init(all_done, 1);
    for (int s = 0; s < ST; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 17) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32((const void*)tmem_slot)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *tmem_slot;
  const uint32_t tS = tmem, tP = tmem + 128, tV = tmem + 256, tK = tmem + 256 + D;
  // this part's share of the walk: `mine` tiles from head `g0` and row tile `n0` on
  const int per_head = *n_needed, total = per_head * group, per = (total + parts.count - 1) / parts.count;
  const int mine = max(0, min(total - part * per, per)), start = next(-1);
  int g0 = 0, n0 = start;
  if (mine > 0) {
    g0 = part * per / per_head;
    for (int skip = part * per % per_head; skip > 0; --skip) n0 = next(n0);
  }

  if (warp < 16) {
    // ------------------------------------------------------------------ scores: a lane a key, 32 of its rows
    const int quarter = warp >> 2, key = k0 + (warp & 3) * 32 + lane;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16, at = lane_base + (uint32_t)(quarter * 32);
    const bool cap = p.cap > 0.f;
    int lo, hi, own = 0;
    rows_of_keys(p, key, key, prefix, lo, hi);
    if (key >= p.Tk) hi = -1;
    if (p.seg_k != nullptr) own = key < p.Tk ? p.seg_k[(long long)b * p.Tk + key] : -1;
    int room = 0;  // dS is worked with times 2^room
    if constexpr (RANGE) {
      float peak = 0.f;
      for (int h = 0; h < group; ++h) peak = fmaxf(peak, sums.peaks[b * p.H + hkv * group + h]);
      room = room_of(peak, sums.peaks[p.B * p.H + b * p.Hkv + hkv]);
    }
    const float up = power_of_two(room), down = power_of_two(-room);
    bool ok = true;
    int it = 0, g = g0, n = n0;
    Score f = score_of(p, hkv * group + g);
    {
      for (; it < mine && ok; ++it) {
        const int q0 = (first + n) * BLK + quarter * 32, stage = it % ST;
        const bool whole = flags[n] & WHOLE;
        uint32_t keep = ~0u;
        if (!whole) {
          keep = span_bits(lo, hi, q0);
          if (p.seg_q != nullptr) keep &= segment_bits(q0 + lane < p.Tq ? p.seg_q[(long long)b * p.Tq + q0 + lane] : -1, own);
        }
        const float* lse = reinterpret_cast<const float*>(smem_raw + C::SUMS + stage * 1024) + quarter * 32;
        ok = mbar_wait(full(stage), (it / ST) & 1, abort_flag) && mbar_wait(s_full, it & 1, abort_flag);
        if (!(ok = __all_sync(0xffffffffu, ok))) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        float x[32], w[32];
        tmem_ld32(tS + at, reinterpret_cast<uint32_t*>(x));
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        probabilities(x, w, f, cap, c_, (float)(key - q0), keep, whole, [&](int e) { return mul_f32x2(*reinterpret_cast<const uint64_t*>(lse + e), both(-1.f)); });
        uint32_t packed[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) packed[e] = pack_16<T>(x[2 * e], x[2 * e + 1]);
        tmem_st16(tS + at, packed);
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(p_ready);
        ok = mbar_wait(dp_full, it & 1, abort_flag);
        if (!(ok = __all_sync(0xffffffffu, ok))) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        tmem_ld32(tP + at, reinterpret_cast<uint32_t*>(x));
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const uint64_t delta2 = *reinterpret_cast<const uint64_t*>(lse + 128 + e);
          const uint64_t dp2 = pack_f32x2(x[e], x[e + 1]);
          const uint64_t past2 = RANGE ? fma_f32x2(delta2, both(-up), mul_f32x2(dp2, both(up))) : fma_f32x2(delta2, both(-1.f), dp2);
          float d0, d1;
          unpack_f32x2(mul_f32x2(past2, pack_f32x2(w[e], w[e + 1])), d0, d1);
          packed[e / 2] = pack_16<T>(d0, d1);
        }
        tmem_st16(tP + at, packed);
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(ds_ready);
        if ((n = next(n)) >= end && it + 1 < mine) {
          n = start;
          f = score_of(p, hkv * group + ++g);
        }
      }
    }
    if (ok && it > 0) {
      ok = __all_sync(0xffffffffu, mbar_wait(all_done, 0, abort_flag));
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    }
    if (ok && parts.count > 1) {
      const long long row = (((long long)b * p.Tk + min(key, p.Tk - 1)) * p.Hkv + hkv) * p.D, size = (long long)p.B * p.Tk * p.Hkv * p.D;
      float* to = parts.sums + (quarter < 2 ? (long long)parts.count * size : 0) + part * size + row;
#pragma unroll 1
      for (int c = (quarter & 1) * (D / 2); c < ((quarter & 1) + 1) * (D / 2); c += 32)
        store_sums(to, (quarter < 2 ? tV : tK) + lane_base + (uint32_t)c, c, p.D, quarter < 2 ? 1.f : down, key < p.Tk, mine == 0);
    } else if (ok) {  // half of the warps store dV, the others dK, each half of the columns
      T* to = (quarter < 2 ? dv : dk) + (((long long)b * p.Tk + min(key, p.Tk - 1)) * p.Hkv + hkv) * p.D;
#pragma unroll 1
      for (int c = (quarter & 1) * (D / 2); c < ((quarter & 1) + 1) * (D / 2); c += 32)
        store_row(to, (quarter < 2 ? tV : tK) + lane_base + (uint32_t)c, c, p.D, quarter < 2 ? 1.f : p.scale * down, key < p.Tk, it == 0);
    } else {
      if (lane == 0 && err) atomicExch(err, 53);
      *abort_flag = 1;
    }
  } else if (warp == 16) {
    // ------------------------------------------------------------------ TMA producer
    if (elect_one() && mine > 0) {
      mbar_expect_tx(kv_bar, 2 * TILE);
#pragma unroll
      for (int c = 0; c < C::CH; ++c) {
        tma_load_4d(sK + c * 16384, &map_k, kv_bar, c * 64, k0, hkv, b);
        tma_load_4d(sV + c * 16384, &map_v, kv_bar, c * 64, k0, hkv, b);
      }
      bool ok = true;
      int it = 0, g = g0, n = n0;
      {
        for (; it < mine; ++it, n = next(n)) {
          if (n >= end) {
            n = start;
            ++g;
          }
          const int h = hkv * group + g;
          const int stage = it % ST, q0 = (first + n) * BLK;
          ok = mbar_wait(empty(stage), ((it / ST) & 1) ^ 1, abort_flag);
          if (!ok) break;
          mbar_expect_tx(full(stage), 2 * TILE + 1024);
          const uint32_t dst = sQG + stage * C::STAGE;
#pragma unroll
          for (int c = 0; c < C::CH; ++c) tma_load_4d(dst + c * 16384, &map_q, full(stage), c * 64, q0, h, b);
#pragma unroll
          for (int c = 0; c < C::CH; ++c) tma_load_4d(dst + TILE + c * 16384, &map_g, full(stage), c * 64, q0, h, b);
          const long long row = ((long long)b * p.H + h) * sums.pitch + q0;
          const uint32_t to = base + C::SUMS + stage * 1024;
          asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], 512, [%2];" ::"r"(to), "l"(sums.lse + row), "r"(full(stage)) : "memory");
          asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], 512, [%2];" ::"r"(to + 512), "l"(sums.delta + row), "r"(full(stage)) : "memory");
        }
      }
      if (!ok) {
        if (err) atomicExch(err, 51);
        *abort_flag = 1;
        for (uint32_t spin = 0; spin < (1u << 16); ++spin)
          if (mbar_try_wait(kv_bar, 0)) break;
        for (int n = max(0, it - ST); n < it; ++n)
          for (uint32_t spin = 0; spin < (1u << 16); ++spin)
            if (mbar_try_wait(full(n % ST), (n / ST) & 1)) break;
      }
    }
  } else {
    // ------------------------------------------------------------------ MMA issuer
    if (elect_one() && mine > 0) {
      constexpr uint32_t idesc_s = product_desc<T>(128, 128, false), idesc_o = product_desc<T>(128, D, true);
      auto rows = [&](uint32_t to, uint32_t a, uint32_t bb) {  // 128 x 128 over the head dimension
#pragma unroll
        for (int c = 0; c < C::CH; ++c) {
          const uint64_t adesc = make_smem_desc(a + c * 16384, false), bdesc = make_smem_desc(bb + c * 16384, false);
#pragma unroll
          for (int k = 0; k < 4; ++k) umma_bf16(to, adesc + (uint64_t)(2 * k), bdesc + (uint64_t)(2 * k), idesc_s, (c > 0 || k > 0) ? 1u : 0u);
        }
      };
      auto cols = [&](uint32_t to, uint32_t a, uint32_t bb, bool add) {  // 128 x D over the 128 rows of the tile at bb
        const uint64_t bdesc = mn_desc(bb, 16384);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          umma_bf16_ts(to, a + (uint32_t)((k >> 1) * 32 + (k & 1) * 8), bdesc + (uint64_t)((2048u >> 4) * k), idesc_o, (add || k > 0) ? 1u : 0u);
      };
      auto q_of = [&](int it) { return sQG + (uint32_t)((it % ST) * C::STAGE); };
      bool ok = mbar_wait(kv_bar, 0, abort_flag) && mbar_wait(full(0), 0, abort_flag);
      if (ok) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        rows(tS, sK, q_of(0));
        umma_commit(s_full);
        rows(tP, sV, q_of(0) + TILE);
        umma_commit(dp_full);
      }
      for (int it = 0; it < mine && ok; ++it) {
        ok = mbar_wait(p_ready, it & 1, abort_flag);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        cols(tV, tS, q_of(it) + TILE, it > 0);
        if (it + 1 < mine) {
          ok = mbar_wait(full((it + 1) % ST), ((it + 1) / ST) & 1, abort_flag);
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          rows(tS, sK, q_of(it + 1));
          umma_commit(s_full);
        }
        ok = mbar_wait(ds_ready, it & 1, abort_flag);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        cols(tK, tP, q_of(it), it > 0);
        umma_commit(empty(it % ST));
        if (it + 1 < mine) {
          rows(tP, sV, q_of(it + 1) + TILE);
          umma_commit(dp_full);
        }
      }
      if (ok) umma_commit(all_done);
      else {
        if (err) atomicExch(err, 52);
        *abort_flag = 1;
      }
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  __syncwarp();
  if (warp == 17) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

// ------------------------------------------------------------------------------------------------ dQ
template <int D>
struct DqCfg {
  // K is read by the first and by the last product of a tile, V by the one between: three places for K and one for V hold as much as
  // two of both, and neither is waited for
  static constexpr int CH = D / 64, TILE = CH * 16384, KS = D == 128 ? 3 : 5, VS = D == 128 ? 1 : 3;
  static constexpr int BARS = (2 + KS + VS) * TILE, FLAGS = BARS + 256;
};

template <typename T, int D>
__global__ void __launch_bounds__(BWD_THREADS, 1)
rules_dq_sm100(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
               const __grid_constant__ CUtensorMap map_g, const Rules p, const Cap c_, const Sums sums, T* dq, int* err) {
  using C = DqCfg<D>;
  constexpr int TILE = C::TILE, KS = C::KS, VS = C::VS;
  constexpr bool RANGE = __is_same(T, __half);
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t base = smem_u32(smem_raw);
  if (base & 1023u) {
    if (threadIdx.x == 0 && err) atomicExch(err, 60);
    return;
  }
  const uint32_t sQ = base, sG = base + TILE, sK = base + 2 * TILE, sV = sK + KS * TILE, bar_base = base + C::BARS;
  uint8_t* flags = smem_raw + C::FLAGS;
  const uint32_t q_bar = bar_base, dp_full = bar_base + 8, ds_ready = bar_base + 16, all_done = bar_base + 24;
  auto s_full = [&](int i) { return bar_base + 32u + 8u * i; };
  auto k_full = [&](int s) { return bar_base + 48u + 8u * s; };
  auto k_empty = [&](int s) { return bar_base + 48u + 8u * (KS + s); };
  auto v_full = [&](int s) { return bar_base + 48u + 8u * (2 * KS + s); };
  auto v_empty = [&](int s) { return bar_base + 48u + 8u * (2 * KS + VS + s); };
  static_assert(48 + 16 * (KS + VS) + 8 <= 256, "barrier area");
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem_raw + C::BARS + 48 + 16 * (KS + VS));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int groups = p.H * p.B, n_q = (p.Tq + BLK - 1) / BLK, q0 = (n_q - 1 - (int)(blockIdx.x / groups)) * BLK;
  const int h = (int)(blockIdx.x % groups) % p.H, b = (int)(blockIdx.x % groups) / p.H, hkv = h / (p.H / p.Hkv);
  const int prefix = prefix_of(p, b);
  int first, last;  // tiles of keys
  keys_of_rows(p, q0, min(q0 + BLK, p.Tq) - 1, prefix, first, last);
  first /= BLK;
  last = last < 0 ? -1 : last / BLK;
  for (int n = threadIdx.x; first + n <= last; n += BWD_THREADS) flags[n] = (uint8_t)tile_flags(p, b, q0, (first + n) * BLK, prefix);
  const int end = last - first + 1;
  auto next = [&](int n) {
    do ++n;
    while (n < end && !(flags[n] & NEEDED));
    return n;
  };
  if (threadIdx.x == 0) {
    mbar_init(q_bar, 1);
    mbar_init(dp_full, 1);
    mbar_init(ds_ready, 16);
    mbar_init(all_done, 1);
    mbar_init(s_full(0), 1);
    mbar_init(s_full(1), 1);
    for (int s = 0; s < KS; ++s) {
      mbar_init(k_full(s), 1);
      mbar_init(k_empty(s), 1);
    }
    for (int s = 0; s < VS; ++s) {
      mbar_init(v_full(s), 1);
      mbar_init(v_empty(s), 1);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 17) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32((const void*)tmem_slot)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *tmem_slot;
  const uint32_t tP = tmem + 256, tQ = tmem + 384;
  const int start = next(-1);

  if (warp < 16) {
    // ------------------------------------------------------------------ scores: a lane a row, 32 of its keys
    const int part = warp >> 2, row = (warp & 3) * 32 + lane, qi = q0 + row;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16, at = lane_base + (uint32_t)(part * 32);
    const bool cap = p.cap > 0.f;
    const Score f = score_of(p, h);
    int lo, hi, own = 0;
    row_span(p, qi, prefix, lo, hi);
    if (qi >= p.Tq) hi = -1;
    if (p.seg_q != nullptr) own = qi < p.Tq ? p.seg_q[(long long)b * p.Tq + qi] : -1;
    const long long sum_at = ((long long)b * p.H + h) * sums.pitch + qi;
    const int room = RANGE ? room_of(sums.peaks[b * p.H + h], sums.peaks[p.B * p.H + b * p.Hkv + hkv]) : 0;  // dS is worked with times 2^room
    const float up = power_of_two(room), down = power_of_two(-room);
    const uint64_t minus_lse2 = both(-sums.lse[sum_at]), minus_delta2 = both(-sums.delta[sum_at] * up), up2 = both(up);
    bool ok = true;
    int it = 0;
    for (int n = start; n < end; n = next(n), ++it) {
      const int k0 = (first + n) * BLK + part * 32;
      const bool whole = flags[n] & WHOLE;
      const uint32_t tS = tmem + (uint32_t)((it & 1) * 128) + at;
      uint32_t keep = ~0u;
      if (!whole) {
        keep = span_bits(lo, hi, k0);
        if (p.seg_k != nullptr) keep &= segment_bits(k0 + lane < p.Tk ? p.seg_k[(long long)b * p.Tk + k0 + lane] : -1, own);
      }
      ok = mbar_wait(s_full(it & 1), (it >> 1) & 1, abort_flag);
      if (!(ok = __all_sync(0xffffffffu, ok))) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      float x[32], w[32];
      tmem_ld32(tS, reinterpret_cast<uint32_t*>(x));
      asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
      probabilities(x, w, f, cap, c_, (float)(qi - k0), keep, whole, [&](int) { return minus_lse2; });
      ok = mbar_wait(dp_full, it & 1, abort_flag);
      if (!(ok = __all_sync(0xffffffffu, ok))) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      tmem_ld32(tP + at, reinterpret_cast<uint32_t*>(x));
      asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
      uint32_t packed[16];
#pragma unroll
      for (int e = 0; e < 32; e += 2) {
        float d0, d1;
        const uint64_t dp2 = pack_f32x2(x[e], x[e + 1]);
        unpack_f32x2(mul_f32x2(RANGE ? fma_f32x2(dp2, up2, minus_delta2) : add_f32x2(dp2, minus_delta2), pack_f32x2(w[e], w[e + 1])), d0, d1);
        packed[e / 2] = pack_16<T>(d0, d1);
      }
      tmem_st16(tS, packed);
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(ds_ready);
    }
    if (ok && it > 0) {
      ok = __all_sync(0xffffffffu, mbar_wait(all_done, 0, abort_flag));
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    }
    if (ok) {  // a quarter of the warps for every 32 columns
      T* to = dq + (((long long)b * p.Tq + min(qi, p.Tq - 1)) * p.H + h) * p.D;
      if (part * 32 < D) store_row(to, tQ + lane_base + (uint32_t)(part * 32), part * 32, p.D, p.scale * down, qi < p.Tq, it == 0);
    } else {
      if (lane == 0 && err) atomicExch(err, 63);
      *abort_flag = 1;
    }
  } else if (warp == 16) {
    // ------------------------------------------------------------------ TMA producer
    if (elect_one() && start < end) {
      mbar_expect_tx(q_bar, 2 * TILE);
#pragma unroll
      for (int c = 0; c < C::CH; ++c) {
        tma_load_4d(sQ + c * 16384, &map_q, q_bar, c * 64, q0, h, b);
        tma_load_4d(sG + c * 16384, &map_g, q_bar, c * 64, q0, h, b);
      }
      bool ok = true;
      int it_k = 0, it_v = 0;
      auto load_k = [&](int n) {
        const int s = it_k % KS;
        if (!mbar_wait(k_empty(s), ((it_k / KS) & 1) ^ 1, abort_flag)) return false;
        mbar_expect_tx(k_full(s), TILE);
#pragma unroll
        for (int c = 0; c < C::CH; ++c) tma_load_4d(sK + s * TILE + c * 16384, &map_k, k_full(s), c * 64, (first + n) * BLK, hkv, b);
        ++it_k;
        return true;
      };
      // in the order of the products: K of a tile goes ahead of V of the tile before
      ok = load_k(start);
      for (int n = start; n < end && ok;) {
        const int then = next(n), s = it_v % VS;
        if (then < end) ok = load_k(then);
        if (ok) ok = mbar_wait(v_empty(s), ((it_v / VS) & 1) ^ 1, abort_flag);
        if (!ok) break;
        mbar_expect_tx(v_full(s), TILE);
#pragma unroll
        for (int c = 0; c < C::CH; ++c) tma_load_4d(sV + s * TILE + c * 16384, &map_v, v_full(s), c * 64, (first + n) * BLK, hkv, b);
        ++it_v;
        n = then;
      }
      if (!ok) {
        if (err) atomicExch(err, 61);
        *abort_flag = 1;
        for (uint32_t spin = 0; spin < (1u << 16); ++spin)
          if (mbar_try_wait(q_bar, 0)) break;
        for (int n = max(0, it_k - KS); n < it_k; ++n)
          for (uint32_t spin = 0; spin < (1u << 16); ++spin)
            if (mbar_try_wait(k_full(n % KS), (n / KS) & 1)) break;
        for (int n = max(0, it_v - VS); n < it_v; ++n)
          for (uint32_t spin = 0; spin < (1u << 16); ++spin)
            if (mbar_try_wait(v_full(n % VS), (n / VS) & 1)) break;
      }
    }
  } else {
    // ------------------------------------------------------------------ MMA issuer
    if (elect_one() && start < end) {
      constexpr uint32_t idesc_s = product_desc<T>(128, 128, false), idesc_o = product_desc<T>(128, D, true);
      auto rows = [&](uint32_t to, uint32_t a, uint32_t bb) {
#pragma unroll
        for (int c = 0; c < C::CH; ++c) {
          const uint64_t adesc = make_smem_desc(a + c * 16384, false), bdesc = make_smem_desc(bb + c * 16384, false);
#pragma unroll
          for (int k = 0; k < 4; ++k) umma_bf16(to, adesc + (uint64_t)(2 * k), bdesc + (uint64_t)(2 * k), idesc_s, (c > 0 || k > 0) ? 1u : 0u);
        }
      };
      auto scores = [&](int it) {
        const int s = it % KS;
        if (!mbar_wait(k_full(s), (it / KS) & 1, abort_flag)) return false;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        rows(tmem + (uint32_t)((it & 1) * 128), sQ, sK + s * TILE);
        umma_commit(s_full(it & 1));
        return true;
      };
      auto grads = [&](int it) {
        const int s = it % VS;
        if (!mbar_wait(v_full(s), (it / VS) & 1, abort_flag)) return false;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        rows(tP, sG, sV + s * TILE);
        umma_commit(dp_full);
        umma_commit(v_empty(s));
        return true;
      };
      int total = 0;
      for (int n = start; n < end; n = next(n)) ++total;
      bool ok = mbar_wait(q_bar, 0, abort_flag) && scores(0) && (total < 2 || scores(1)) && grads(0);
      for (int it = 0; it < total && ok; ++it) {
        ok = mbar_wait(ds_ready, it & 1, abort_flag);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint64_t bdesc = mn_desc(sK + (it % KS) * TILE, 16384);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          umma_bf16_ts(tQ, tmem + (uint32_t)((it & 1) * 128 + (k >> 1) * 32 + (k & 1) * 8), bdesc + (uint64_t)((2048u >> 4) * k), idesc_o, (it > 0 || k > 0) ? 1u : 0u);
        umma_commit(k_empty(it % KS));
        if (it + 1 < total) ok = grads(it + 1);
        if (ok && it + 2 < total) ok = scores(it + 2);
      }
      if (ok) umma_commit(all_done);
      else {
        if (err) atomicExch(err, 62);
        *abort_flag = 1;
      }
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  __syncwarp();
  if (warp == 17) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

// Parts that a key tile's walk is split into: with fewer key tiles than SMs (few key heads, whose query heads are all walked over one after the other),
// as many as fill the chip, of four tiles each at least.  A part of its own costs its start, about three tiles, and its sums in memory.
int parts_of(int B, int H, int Hkv, int Tq, int Tk) {
  const long long units = (long long)((Tk + BLK - 1) / BLK) * Hkv * B, sms = kb_sm_count();
  const long long walk = (long long)(H / Hkv) * ((Tq + BLK - 1) / BLK);
  if (units >= sms) return 1;
  const long long want = (sms + units - 1) / units, most = walk / 4;
  return (int)std::max(1ll, std::min(std::min(want, most), 16ll));
}

int flag_bytes(int T) { return ((T + BLK - 1) / BLK + 15) / 16 * 16; }

template <typename T, int D>
int launch_bwd(const CUtensorMap* m, const Rules& p, const Sums& sums, void* dq, void* dk, void* dv, const Parts& parts, int* err, cudaStream_t stream) {
  static bool attr[2][KB_MAX_DEVICES] = {{false}};
  if (!kb_allow_smem(rules_dkv_sm100<T, D>, DkvCfg<D>::FLAGS + MAX_BLOCKS, attr[0]) || !kb_allow_smem(rules_dq_sm100<T, D>, DqCfg<D>::FLAGS + MAX_BLOCKS, attr[1])) {
    kb200_set_error("attention_rules: shared-memory limit");
    return -3;
  }
  const Cap cap = make_cap(p.scale, p.cap);
  if (dk != nullptr)
    rules_dkv_sm100<T, D><<<(unsigned)((long long)((p.Tk + BLK - 1) / BLK) * p.Hkv * p.B * parts.count), BWD_THREADS, DkvCfg<D>::FLAGS + flag_bytes(p.Tq), stream>>>(m[0], m[1], m[2], m[3], p, cap,
                                                                                                                                               sums, (T*)dk, (T*)dv, parts, err);
  if (dk != nullptr && parts.count > 1) {
    const long long n = (long long)p.B * p.Tk * p.Hkv * p.D / 4;
    join_parts_kernel<T><<<(unsigned)((2 * n + 255) / 256), 256, 0, stream>>>((const float4*)parts.sums, (T*)dk, (T*)dv, parts.count, n, p.scale);
  }
  if (dq != nullptr)
    rules_dq_sm100<T, D><<<(unsigned)((long long)((p.Tq + BLK - 1) / BLK) * p.H * p.B), BWD_THREADS, DqCfg<D>::FLAGS + flag_bytes(p.Tk), stream>>>(m[0], m[1], m[2], m[3], p, cap, sums,
                                                                                                                                           (T*)dq, err);
  return 0;
}

}  // namespace

// Floats of workspace that kb200_attention_rules_bwd_sm100 takes for dk and dv at these sizes.
KB_API long long kb200_attention_rules_bwd_work(int B, int H, int Hkv, int Tq, int Tk, int D) {
  if (B <= 0 || Hkv <= 0 || H < Hkv || Tq <= 0 || Tk <= 0 || D <= 0) return 0;
  const int parts = parts_of(B, H, Hkv, Tq, Tk);
  return parts > 1 ? 2ll * parts * B * Tk * Hkv * D : 0;
}

// As kb200_attention_rules_bwd for what kb200_attention_rules_fwd_sm100 takes, at most 1048576 rows and keys; lse and delta with rows `pitch` apart, a
// multiple of 128.  peaks: float16 B * (H + Hkv) floats of workspace, bfloat16 null.  work: `floats` of them, 16-byte aligned, as many as
// kb200_attention_rules_bwd_work says, or null.
KB_API int kb200_attention_rules_bwd_sm100(const void* q, const void* k, const void* v, const void* grad_out, const long long* strides, const float* lse, const float* delta,
                                           int pitch, float* peaks, void* dq, void* dk, void* dv, int dtype, int B, int H, int Hkv, int Tq, int Tk, int D, int* err, float* work, long long floats, float scale, float cap,
                                           const float* slopes, int causal, int window, const int* prefix, const int* seg_q, const int* seg_k, const void* range_q,
                                           const void* range_k, cudaStream_t stream) {
  const Rules p{B, H, Hkv, Tq, Tk, D, scale, cap, slopes, causal, window, prefix, seg_q, seg_k, (const int4*)range_q, (const int4*)range_k};
  if (B <= 0 || H <= 0 || Hkv <= 0 || H % Hkv || Tq <= 0 || Tk <= 0 || D <= 0 || D > 128 || D % 8 || (dtype != 1 && dtype != 2) || Tk > MAX_BLOCKS * BLK ||
      Tq > MAX_BLOCKS * BLK || pitch % BLK || pitch < Tq || (long long)((Tq + 127) / 128) * H * B > 0x7fffffffll || (long long)((Tk + 127) / 128) * Hkv * B > 0x7fffffffll) {
    kb200_set_error("attention_rules_bwd_sm100: sizes out of range");
    return -2;
  }
  const Strides qs{strides[0], strides[1], strides[2]}, ks{strides[3], strides[4], strides[5]}, vs{strides[6], strides[7], strides[8]}, gs{strides[9], strides[10], strides[11]};
  if (!rules_strides(qs, q, Tq, H, B) || !rules_strides(ks, k, Tk, Hkv, B) || !rules_strides(vs, v, Tk, Hkv, B) || !rules_strides(gs, grad_out, Tq, H, B) ||
      (((uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv | (uintptr_t)lse | (uintptr_t)delta) & 15)) {
    kb200_set_error("attention_rules_bwd_sm100: strides and base pointers must be multiples of 16 bytes");
    return -2;
  }
  const bool half = dtype == 2;
  if (half && peaks == nullptr) {
    kb200_set_error("attention_rules_bwd_sm100: float16 needs a workspace for its rows' norms");
    return -2;
  }
  CUtensorMap m[4];
  if (!rules_map(&m[0], q, D, Tq, H, B, qs, 128, half) || !rules_map(&m[1], k, D, Tk, Hkv, B, ks, 128, half) || !rules_map(&m[2], v, D, Tk, Hkv, B, vs, 128, half) ||
      !rules_map(&m[3], grad_out, D, Tq, H, B, gs, 128, half)) {
    kb200_set_error("attention_rules_bwd_sm100: cuTensorMapEncodeTiled failed");
    return -3;
  }
  const Sums sums{lse, delta, pitch, peaks};
  if (half) launch_peaks((const __half*)grad_out, gs, (const __half*)v, vs, peaks, p, stream);
  Parts parts{parts_of(B, H, Hkv, Tq, Tk), work};
  if (work == nullptr || 2ll * parts.count * B * Tk * Hkv * D > floats) parts.count = 1;
  int rc;
  if (D <= 64) rc = half ? launch_bwd<__half, 64>(m, p, sums, dq, dk, dv, parts, err, stream) : launch_bwd<__nv_bfloat16, 64>(m, p, sums, dq, dk, dv, parts, err, stream);
  else rc = half ? launch_bwd<__half, 128>(m, p, sums, dq, dk, dv, parts, err, stream) : launch_bwd<__nv_bfloat16, 128>(m, p, sums, dq, dk, dv, parts, err, stream);
  if (rc != 0) return rc;
  KB_CHECK_LAUNCH("attention_rules_bwd_sm100");
  return 0;
}

KB_API int kb200_attention_rules_delta(const void* o, const void* lo, const void* grad_out, const long long* strides, float* delta, int pitch, int dtype, int B, int H, int Tq, int D,
                                       cudaStream_t stream);

// All of a gradient in one call: delta, from o, lo (may be null) and grad_out, then the above.  delta: B * H * pitch floats, and float16 B * (H + Hkv) more
// behind them for the norms.
KB_API int kb200_attention_rules_grads_sm100(const void* q, const void* k, const void* v, const void* o, const void* lo, const void* grad_out, const long long* strides,
                                             const float* lse, float* delta, int pitch, void* dq, void* dk, void* dv, int dtype, int B, int H, int Hkv, int Tq, int Tk, int D, int* err,
                                             float* work, long long floats, float scale, float cap, const float* slopes, int causal, int window, const int* prefix, const int* seg_q, const int* seg_k,
                                             const void* range_q, const void* range_k, cudaStream_t stream) {
  const int rc = kb200_attention_rules_delta(o, lo, grad_out, strides + 9, delta, pitch, dtype, B, H, Tq, D, stream);
  return rc != 0 ? rc
                 : kb200_attention_rules_bwd_sm100(q, k, v, grad_out, strides, lse, delta, pitch, dtype == 2 ? delta + (long long)B * H * pitch : nullptr, dq, dk, dv, dtype, B, H, Hkv, Tq, Tk, D, err, work, floats, scale, cap, slopes, causal, window, prefix,
                                                   seg_q, seg_k, range_q, range_k, stream);
}
