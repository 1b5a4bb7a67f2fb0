// What the attention kernels with scores by rule share: the score of a pair, which keys a row sees, and which tiles can be left out.
//
//   s(i, j) = scale * q_i . k_j,   with a cap c: c * tanh(s / c),   with slopes: less slope_h * |i - j|
//   row i sees key j when all of these hold
//     causal   j <= i, or j < prefix_b
//     window   |i - j| < window
//     segments seg_q(b, i) == seg_k(b, j) >= 0
// The first two give each row one span [lo, hi] of keys; segments (ids in any order) are compared pair by pair.  A row that sees nothing
// is zero, and so is its gradient.
#pragma once
#include <cuda_fp16.h>
#include <limits.h>

#include "common.cuh"

namespace kbrules {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int SEG_TILE = 128;  // positions whose ids one entry of the segment ranges stands for

struct Rules {
  int B, H, Hkv, Tq, Tk, D;
  float scale;
  float cap;            // 0: none
  const float* slopes;  // [H] or null
  int causal, window;   // window 0: none
  const int* prefix;    // [B] or null (with causal)
  const int *seg_q, *seg_k;  // [B, Tq], [B, Tk] contiguous, or null
  const int4 *range_q, *range_k;  // per SEG_TILE positions: lowest id, highest id, any negative id, -
};

// Strides in elements; the head dimension has unit stride.
struct Strides {
  long long t, h, b;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// tanh(x) for |x| <= 1: x times a polynomial of degree 6 in x^2 (a linear program over 3000 Chebyshev points for the least maximum relative
// error, 5e-8; 1.7e-7 in float32).  Scores stay below their cap as a rule, so that this is what runs: seven instructions on the FMA
// pipe instead of an exponential and a reciprocal on the one that the softmax needs.  A NaN stays one.
__device__ __forceinline__ float tanh_small(float x) {
  const float u = x * x;
  float p = 0.0010410323739051819f;
  p = fmaf(p, u, -0.0062033990398049355f);
  p = fmaf(p, u, 0.020289991050958633f);
  p = fmaf(p, u, -0.05345702916383743f);
  p = fmaf(p, u, 0.13325203955173492f);
  p = fmaf(p, u, -0.33332839608192444f);
  p = fmaf(p, u, 0.9999999403953552f);
  return p * x;
}
// Any x: beyond 1 as 1 - 2 / (1 + e^(2x)), which loses nothing there.
__device__ __forceinline__ float tanh_any(float x) {
  const float a = fabsf(x);
  if (a <= 1.f) return tanh_small(x);
  const float t = 1.f - __fdividef(2.f, 1.f + ex2(fminf(a, 32.f) * (2.f * LOG2E)));
  return x != x ? x : copysignf(t, x);
}

// Factors of one head's scores; results are in units of log2, as the exponentials take them.
struct Score {
  float pre, post;  // no cap: s * post; cap: tanh(s * pre) * post
  float slope;      // of |i - j|, in log2
};
__device__ __forceinline__ Score score_of(const Rules& r, int h) {
  Score s;
  s.pre = r.cap > 0.f ? r.scale / r.cap : 1.f;
  s.post = (r.cap > 0.f ? r.cap : r.scale) * LOG2E;
  s.slope = r.slopes != nullptr ? r.slopes[h] * LOG2E : 0.f;
  return s;
}

// Keys that a causal mask does not hide; less than none is none (the lowest number less one would wrap around).
__device__ __forceinline__ int prefix_of(const Rules& r, int b) { return r.prefix != nullptr ? max(r.prefix[b], 0) : 0; }

__device__ __forceinline__ void row_span(const Rules& r, int i, int prefix, int& lo, int& hi) {
  lo = 0;
  hi = r.Tk - 1;
  if (r.causal) hi = min(hi, max(i, prefix - 1));
  if (r.window > 0) {
    lo = max(0, i - r.window + 1);
    hi = min(hi, i + r.window - 1);
  }
}
// Keys that any of the rows [i0, i1] may see, and rows that may see any of the keys [k0, k1].
__device__ __forceinline__ void keys_of_rows(const Rules& r, int i0, int i1, int prefix, int& lo, int& hi) {
  int unused;
  row_span(r, i0, prefix, lo, unused);
  row_span(r, i1, prefix, unused, hi);
}
__device__ __forceinline__ void rows_of_keys(const Rules& r, int k0, int k1, int prefix, int& lo, int& hi) {
  lo = r.causal && k0 >= prefix ? k0 : 0;
  hi = r.Tq - 1;
  if (r.window > 0) {
    lo = max(lo, k0 - r.window + 1);
    hi = min(hi, k1 + r.window - 1);
  }
}
// Whether segments leave anything of rows [i0, i1] against keys [k0, k1]; both lie within one entry of the ranges each.
__device__ __forceinline__ int n_ranges(int T) { return (T + SEG_TILE - 1) / SEG_TILE; }
__device__ __forceinline__ bool segments_meet(const Rules& r, int b, int i0, int k0) {
  if (r.seg_q == nullptr) return true;
  const int4 a = r.range_q[(long long)b * n_ranges(r.Tq) + i0 / SEG_TILE], c = r.range_k[(long long)b * n_ranges(r.Tk) + k0 / SEG_TILE];
  return a.x <= c.y && c.x <= a.y;
}
// Whether they let every row of the one see every key of the other.
__device__ __forceinline__ bool segments_same(const Rules& r, int b, int i0, int k0) {
  if (r.seg_q == nullptr) return true;
  const int4 a = r.range_q[(long long)b * n_ranges(r.Tq) + i0 / SEG_TILE], c = r.range_k[(long long)b * n_ranges(r.Tk) + k0 / SEG_TILE];
  return a.x == a.y && c.x == c.y && a.x == c.x && a.z == 0 && c.z == 0;
}

template <typename T>
__device__ __forceinline__ float load_f32(const T* p) {
  return to_f32<T>(*p);
}

}  // namespace kbrules

template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
