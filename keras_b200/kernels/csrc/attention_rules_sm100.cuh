// What the tensor-core kernels of attention by rules share: which tiles of 128 x 128 pairs have to be looked at, and the scores of a thread's
// part of one.  attention_rules.cuh says what a score is and which keys a row sees.
#pragma once
#include "attention_rules.cuh"
#include "attention_sm100.cuh"

namespace kbrules {
using namespace kbgemm;
using namespace kbattn;

constexpr int BLK = 128;
constexpr int MAX_BLOCKS = 8192;  // tiles of keys (or rows) that one CTA's flags hold: 1048576 positions
enum { NEEDED = 1, WHOLE = 2 };   // flags of a pair of tiles: some pair is visible; every pair is

// Flags of rows i0 .. i0 + 127 against keys k0 .. k0 + 127.
__device__ __forceinline__ int tile_flags(const Rules& r, int b, int i0, int k0, int prefix) {
  const int i1 = min(i0 + BLK, r.Tq) - 1, k1 = min(k0 + BLK, r.Tk) - 1;
  if (i1 < i0 || k1 < k0) return 0;
  int lo, hi;
  keys_of_rows(r, i0, i1, prefix, lo, hi);
  if (k0 > hi || k1 < lo || !segments_meet(r, b, i0, k0)) return 0;
  bool whole = k0 + BLK <= r.Tk && segments_same(r, b, i0, k0);
  if (r.causal && k1 > i0 && k1 >= prefix) whole = false;
  if (r.window > 0 && (i1 - k0 >= r.window || k1 - i0 >= r.window)) whole = false;
  return NEEDED | (whole ? WHOLE : 0);
}

__device__ __forceinline__ uint64_t mul_f32x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t both(float a) { return pack_f32x2(a, a); }

// The cap of a call as the kernels take it: tanh(s * pre) * post from polynomials in x^2 = (s * pre)^2 whose coefficients hold `post` already.
struct Cap {
  float pre, post, inv_post;
  float near[4], far[6];
  float mid_raw[5];   // of x = s itself
  bool folds;         // they are all well within the type
};
// tanh(x) / x for |x| <= 1/2 (degree 3 in x^2), 3/4 (degree 4) and 1 (degree 5), fitted as tanh_small's: 5.4e-7 to 5.9e-7 of the value, a thousandth of what rounding
// the probabilities to 16 bits costs under a cap of 50.  As a rule scores stay below half of their cap, and tanh is six instructions on the
// FMA pipe instead of an exponential and a reciprocal on the one that the softmax needs.
static inline Cap make_cap(float scale, float cap) {
  const float near[4] = {0.999999463558197f, -0.33326318860054016f, 0.13190299272537231f, -0.04440227895975113f};
  const float far[6] = {0.9999994039535522f, -0.3332904279232025f, 0.13281434774398804f, -0.051605693995952606f, 0.016743140295147896f, -0.0030670708511024714f};
  const double mid[5] = {0.999999463558197, -0.3332825005054474, 0.13258983194828033, -0.050056297332048416, 0.012929627671837807};
  Cap c{};
  if (cap > 0.f) {
    c.pre = scale / cap;
    c.post = cap * LOG2E;
    c.inv_post = 1.f / c.post;
    for (int i = 0; i < 4; ++i) c.near[i] = near[i] * c.post;
    for (int i = 0; i < 6; ++i) c.far[i] = far[i] * c.post;
    const double a = fabs((double)c.pre);
    c.folds = a > 1e-4 && a < 1e3 && cap > 1e-6f && cap < 1e6f;
    if (c.folds)
      for (int i = 0; i < 5; ++i) c.mid_raw[i] = (float)(mid[i] * (double)c.post * pow((double)c.pre, 2 * i + 1));
  }
  return c;
}

// 32 raw scores to tanh(s * pre) * post, for a warp, by the shortest form that all its lanes allow.
__device__ __forceinline__ void capped(float (&x)[32], const Cap& c) {
  const uint64_t pre2 = both(c.pre);
  float top = 0.f;
#pragma unroll
  for (int e = 0; e < 32; e += 2) {
    unpack_f32x2(mul_f32x2(pack_f32x2(x[e], x[e + 1]), pre2), x[e], x[e + 1]);
    top = fmaxf(fmaxf(top, fabsf(x[e])), fabsf(x[e + 1]));
  }
  if (!__any_sync(0xffffffffu, top > 0.5f)) {
    const uint64_t a0 = both(c.near[0]), a1 = both(c.near[1]), a2 = both(c.near[2]), a3 = both(c.near[3]);
#pragma unroll
    for (int e = 0; e < 32; e += 2) {
      const uint64_t v = pack_f32x2(x[e], x[e + 1]), u = mul_f32x2(v, v);
      unpack_f32x2(mul_f32x2(fma_f32x2(fma_f32x2(fma_f32x2(a3, u, a2), u, a1), u, a0), v), x[e], x[e + 1]);
    }
  } else if (!__any_sync(0xffffffffu, top > 1.f)) {
    const uint64_t a0 = both(c.far[0]), a1 = both(c.far[1]), a2 = both(c.far[2]), a3 = both(c.far[3]), a4 = both(c.far[4]), a5 = both(c.far[5]);
#pragma unroll
    for (int e = 0; e < 32; e += 2) {
      const uint64_t v = pack_f32x2(x[e], x[e + 1]), u = mul_f32x2(v, v);
      unpack_f32x2(mul_f32x2(fma_f32x2(fma_f32x2(fma_f32x2(fma_f32x2(fma_f32x2(a5, u, a4), u, a3), u, a2), u, a1), u, a0), v), x[e], x[e + 1]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 32; ++e) x[e] = tanh_any(x[e]) * c.post;
  }
}
// 32 raw scores to scores in log2; `from` - e is the distance of the pair.  A score that is not capped is multiplied with `post`.
__device__ __forceinline__ void scores32(float (&x)[32], bool cap, const Cap& c, float post, float slope, float from) {
  if (cap) capped(x, c);
  else if (post != 1.f) {
#pragma unroll
    for (int e = 0; e < 32; ++e) x[e] *= post;
  }
  if (slope != 0.f) {
#pragma unroll
    for (int e = 0; e < 32; ++e) x[e] = fmaf(-slope, fabsf(from - (float)e), x[e]);
  }
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Bits of the elements e of 32 with lo <= at + e <= hi.
__device__ __forceinline__ uint32_t span_bits(int lo, int hi, int at) {
  const int a = lo - at, z = hi - at;
  if (z < 0 || a > 31 || z < a) return 0;
  return (0xffffffffu >> (31 - min(z, 31))) & (0xffffffffu << max(a, 0));
}
// Bits of the elements whose segment is the lane's own; `id`: the segment of element `lane`.
__device__ __forceinline__ uint32_t segment_bits(int id, int own) {
  const int lo = __reduce_min_sync(0xffffffffu, id), hi = __reduce_max_sync(0xffffffffu, id);
  if (lo == hi) return lo == own && own >= 0 ? 0xffffffffu : 0u;
  uint32_t bits = 0;
#pragma unroll
  for (int e = 0; e < 32; ++e) bits |= (__shfl_sync(0xffffffffu, id, e) == own ? 1u : 0u) << e;
  return own >= 0 ? bits : 0u;
}

template <typename T>
__device__ __forceinline__ uint32_t pack_16(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack_16<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack_16<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <typename T>
__device__ __forceinline__ void unpack_16(uint32_t w, float& a, float& b);
template <>
__device__ __forceinline__ void unpack_16<__nv_bfloat16>(uint32_t w, float& a, float& b) {
  a = __uint_as_float(w << 16);
  b = __uint_as_float(w & 0xffff0000u);
}
template <>
__device__ __forceinline__ void unpack_16<__half>(uint32_t w, float& a, float& b) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  a = f.x;
  b = f.y;
}

// Instruction descriptor of a product of 16-bit operands with float32 sums: M x N, B's major direction.
template <typename T>
constexpr uint32_t product_desc(int m, int n, bool b_mn_major) {
  const uint32_t bf16 = sizeof(T) == 2 && __is_same(T, __nv_bfloat16) ? 1u : 0u;
  return (1u << 4) | (bf16 << 7) | (bf16 << 10) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// Operand of rows of 64 values (128 bytes, swizzled), read along the rows' direction; the next 64 values `next` bytes further.
__device__ __forceinline__ uint64_t mn_desc(uint32_t addr, uint32_t next) {
  return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(next >> 4) << 16) | ((uint64_t)(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// Tensor map of a [B, T, H, D] tensor; a dimension of one element has no stride to speak of.
static inline bool rules_map(CUtensorMap* map, const void* p, int D, int T, int H, int B, const Strides& s, int box_t, bool half) {
  return make_map_bthd(map, p, D, T, H, B, T == 1 ? 8 : s.t, H == 1 ? 8 : s.h, B == 1 ? 8 : s.b, 64, box_t, half);
}
static inline bool rules_strides(const Strides& s, const void* p, int T, int H, int B) {
  auto ok = [](long long v, int n) { return n == 1 || (v > 0 && v % 8 == 0 && v < (1ll << 38)); };
  return ok(s.t, T) && ok(s.h, H) && ok(s.b, B) && ((uintptr_t)p & 15) == 0;
}

}  // namespace kbrules
