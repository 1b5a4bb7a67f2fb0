// Attention with scores by rule, every type and layout: forward pass and gradients on the FMA pipes (attention_rules.cuh says what a score
// is and which keys a row sees).  float32 runs here, and 16-bit tensors that the tensor-core kernels do not take (heads wider than 128,
// strides that are no multiple of 16 bytes).
//
// Forward: a CTA takes BT rows of one head and walks over the tiles of BT keys that any of them may see, with the running maximum and sum
// of the softmax; scores never leave shared memory.  It keeps for each row L = max + log2(sum), from which the gradients get the
// probabilities back as 2^(x - L):
//   dP = dO V^T,  delta_i = sum_d dO_id O_id,  dS = P (dP - delta) (1 - tanh^2),  dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO
// Gradients take two kernels, one a tile of keys (over all rows and all query heads of its group) and one a tile of rows: seven products
// instead of five, but each sum is made by one thread in one order, so that they repeat bit for bit.  Few key tiles are shared out to several blocks,
// whose sums a second launch adds up in order (float32 2 x 1024 x 8/2 x 128: dk and dv 1141 -> 277 us).
//
// What bounds it: 64 multiply-adds a thread for eight 16-byte reads of shared memory, and loads that are waited for: float32 at 4 x 1024 x 12 x 64 takes
// 244 us forward (26 TFLOP/s of the FMA pipes' 75), 429 us dk and dv, 320 us dq (30); at 4 x 333 x 8 x 64 51, 66 and 61 us, where the longest rows' blocks
// alone are what lasts.
#include "attention_rules.cuh"

namespace {
using namespace kbrules;

template <typename T, int DP, int BT>
struct Tile {
  static constexpr int PITCH = DP + 4;  // rows 4 banks apart: eight threads read 16 bytes each of eight rows without a conflict
  static constexpr int FLOATS = BT * PITCH;
  static constexpr int SP = BT + 4;
};

// Rows t0.. of a [T, D] slice into shared memory as float32, zeros beyond the last row and the last column.
template <typename T, int DP, int BT>
__device__ __forceinline__ void load_tile(float* dst, const T* src, long long stride_t, int t0, int n_rows, int D, bool vec) {
  using C = Tile<T, DP, BT>;
  if (vec) {
    constexpr int V = 16 / sizeof(T);
    for (int e = threadIdx.x; e < BT * (DP / V); e += 256) {
      const int r = e / (DP / V), c = (e % (DP / V)) * V;
      uint4 w = make_uint4(0, 0, 0, 0);
      if (t0 + r < n_rows && c < D) w = *reinterpret_cast<const uint4*>(src + (long long)(t0 + r) * stride_t + c);
      const T* t = reinterpret_cast<const T*>(&w);
#pragma unroll
      for (int i = 0; i < V; i += 4)
        *reinterpret_cast<float4*>(dst + r * C::PITCH + c + i) = make_float4(to_f32<T>(t[i]), to_f32<T>(t[i + 1]), to_f32<T>(t[i + 2]), to_f32<T>(t[i + 3]));
    }
  } else {
    for (int e = threadIdx.x; e < BT * DP; e += 256) {
      const int r = e / DP, c = e % DP;
      dst[r * C::PITCH + c] = t0 + r < n_rows && c < D ? load_f32(src + (long long)(t0 + r) * stride_t + c) : 0.f;
    }
  }
}

// acc[i][j] = sum_d a[ty + 16 i][d] * b[tx + 16 j][d]
template <int DP, int M, int PITCH>
__device__ __forceinline__ void product_rows(float (&acc)[M][M], const float* a, const float* b, int ty, int tx) {
#pragma unroll
  for (int i = 0; i < M; ++i)
#pragma unroll
    for (int j = 0; j < M; ++j) acc[i][j] = 0.f;
#pragma unroll 4
  for (int d = 0; d < DP; d += 4) {
    float4 x[M], y[M];
#pragma unroll
    for (int i = 0; i < M; ++i) x[i] = *reinterpret_cast<const float4*>(a + (ty + 16 * i) * PITCH + d);
#pragma unroll
    for (int j = 0; j < M; ++j) y[j] = *reinterpret_cast<const float4*>(b + (tx + 16 * j) * PITCH + d);
#pragma unroll
    for (int i = 0; i < M; ++i)
#pragma unroll
      for (int j = 0; j < M; ++j)
        acc[i][j] = fmaf(x[i].x, y[j].x, fmaf(x[i].y, y[j].y, fmaf(x[i].z, y[j].z, fmaf(x[i].w, y[j].w, acc[i][j]))));
  }
}
// acc[i][4 jj ..] += sum_c s[ty + 16 i][c] * b[c][tx * 4 + 64 jj ..]
template <int DP, int BT, int M, int PITCH, int SP>
__device__ __forceinline__ void product_cols(float (&acc)[M][DP / 16], const float* s, const float* b, int ty, int tx) {
#pragma unroll 2
  for (int c = 0; c < BT; c += 4) {
    float4 w[M];
#pragma unroll
    for (int i = 0; i < M; ++i) w[i] = *reinterpret_cast<const float4*>(s + (ty + 16 * i) * SP + c);
#pragma unroll
    for (int cc = 0; cc < 4; ++cc)
#pragma unroll
      for (int jj = 0; jj < DP / 64; ++jj) {
        const float4 y = *reinterpret_cast<const float4*>(b + (c + cc) * PITCH + tx * 4 + 64 * jj);
#pragma unroll
        for (int i = 0; i < M; ++i) {
          const float x = cc == 0 ? w[i].x : cc == 1 ? w[i].y : cc == 2 ? w[i].z : w[i].w;
          acc[i][4 * jj] = fmaf(x, y.x, acc[i][4 * jj]);
          acc[i][4 * jj + 1] = fmaf(x, y.y, acc[i][4 * jj + 1]);
          acc[i][4 * jj + 2] = fmaf(x, y.z, acc[i][4 * jj + 2]);
          acc[i][4 * jj + 3] = fmaf(x, y.w, acc[i][4 * jj + 3]);
        }
      }
  }
}
template <typename T, int DP, int M>
__device__ __forceinline__ void store_rows(T* out, long long stride_t, const float (&acc)[M][DP / 16], const float (&factor)[M], int t0, int n_rows, int D, int ty, int tx) {
#pragma unroll
  for (int i = 0; i < M; ++i) {
    const int t = t0 + ty + 16 * i;
    if (t >= n_rows) continue;
#pragma unroll
    for (int jj = 0; jj < DP / 64; ++jj)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = tx * 4 + 64 * jj + e;
        if (d < D) out[(long long)t * stride_t + d] = from_f32<T>(acc[i][4 * jj + e] * factor[i]);
      }
  }
}

// A pair's score in log2, and what its derivative by the plain score is multiplied with.
__device__ __forceinline__ float rule_score(const Rules& r, const Score& f, float s, int i, int j, float& through) {
  through = 1.f;
  float x = s * f.post;
  if (r.cap > 0.f) {
    const float t = tanh_any(s * f.pre);
    through = fmaf(-t, t, 1.f);
    x = t * f.post;
  }
  return fmaf(-f.slope, (float)abs(i - j), x);
}

struct Gradients {
  const void* grad_out;
  Strides go;
  const float *lse, *delta;  // [B, H, pitch]
  int pitch;
};

template <typename T, int DP, int BT>
__global__ void __launch_bounds__(256) rules_fwd_kernel(const Rules r, const T* q, Strides qs, const T* k, Strides ks, const T* v, Strides vs, T* o, float* lse, int pitch, int vec) {
  using C = Tile<T, DP, BT>;
  constexpr int M = BT / 16;
  extern __shared__ __align__(16) float sm[];
  float *sQ = sm, *sK = sQ + C::FLOATS, *sV = sK + C::FLOATS, *sP = sV + C::FLOATS;
  const int heads = r.H * r.B, n_q = (r.Tq + BT - 1) / BT;
  const int q0 = (n_q - 1 - (int)(blockIdx.x / heads)) * BT;  // the longest rows of a causal mask first
  const int h = (int)(blockIdx.x % heads) % r.H, b = (int)(blockIdx.x % heads) / r.H, hkv = h / (r.H / r.Hkv);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const T* kb = k + b * ks.b + hkv * ks.h;
  const T* vb = v + b * vs.b + hkv * vs.h;
  load_tile<T, DP, BT>(sQ, q + b * qs.b + h * qs.h, qs.t, q0, r.Tq, r.D, vec & 1);
  const Score f = score_of(r, h);
  const int prefix = prefix_of(r, b);
  int lo[M], hi[M], seg[M], first, last;
  float m[M], l[M], acc[M][DP / 16];
  keys_of_rows(r, q0, min(q0 + BT, r.Tq) - 1, prefix, first, last);
#pragma unroll
  for (int i = 0; i < M; ++i) {
    const int t = q0 + ty + 16 * i;
    row_span(r, t, prefix, lo[i], hi[i]);
    seg[i] = r.seg_q != nullptr && t < r.Tq ? r.seg_q[(long long)b * r.Tq + t] : 0;
    if (t >= r.Tq || seg[i] < 0) hi[i] = -1;
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int e = 0; e < DP / 16; ++e) acc[i][e] = 0.f;
  }
  for (int k0 = first / BT * BT; k0 <= last; k0 += BT) {
    if (!segments_meet(r, b, q0, k0)) continue;
    __syncthreads();
    load_tile<T, DP, BT>(sK, kb, ks.t, k0, r.Tk, r.D, vec & 2);
    load_tile<T, DP, BT>(sV, vb, vs.t, k0, r.Tk, r.D, vec & 4);
    __syncthreads();
    float s[M][M];
    product_rows<DP, M, C::PITCH>(s, sQ, sK, ty, tx);
    int seg_k[M];
#pragma unroll
    for (int j = 0; j < M; ++j) seg_k[j] = r.seg_k != nullptr && k0 + tx + 16 * j < r.Tk ? r.seg_k[(long long)b * r.Tk + k0 + tx + 16 * j] : 0;
#pragma unroll
    for (int i = 0; i < M; ++i) {
      const int t = q0 + ty + 16 * i;
      float top = -INFINITY;
      bool bad = false;  // a NaN among the scores: the maximum alone would pass over it
#pragma unroll
      for (int j = 0; j < M; ++j) {
        const int key = k0 + tx + 16 * j;
        float unused;
        s[i][j] = key >= lo[i] && key <= hi[i] && (r.seg_k == nullptr || seg_k[j] == seg[i]) ? rule_score(r, f, s[i][j], t, key, unused) : -INFINITY;
        top = fmaxf(top, s[i][j]);
        bad |= s[i][j] != s[i][j];
      }
#pragma unroll
      for (int w = 8; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
      const float m_new = fmaxf(m[i], top), base = m_new == -INFINITY ? 0.f : m_new, alpha = ex2(m[i] - base);
      float sum = bad ? NAN : 0.f;
#pragma unroll
      for (int j = 0; j < M; ++j) {
        const float p = ex2(s[i][j] - base);
        sum += p;
        sP[(ty + 16 * i) * C::SP + tx + 16 * j] = p;
      }
#pragma unroll
      for (int w = 8; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
      l[i] = fmaf(l[i], alpha, sum);
      m[i] = m_new;
#pragma unroll
      for (int e = 0; e < DP / 16; ++e) acc[i][e] *= alpha;
    }
    __syncwarp();  // a row's probabilities are written and read by the same half of a warp
    product_cols<DP, BT, M, C::PITCH, C::SP>(acc, sP, sV, ty, tx);
  }
  float inv[M];
#pragma unroll
  for (int i = 0; i < M; ++i) {
    inv[i] = l[i] == 0.f ? 0.f : 1.f / l[i];
    const int t = q0 + ty + 16 * i;
    if (lse != nullptr && tx == 0 && t < r.Tq) lse[((long long)b * r.H + h) * pitch + t] = l[i] == 0.f ? INFINITY : m[i] + log2f(l[i]);
  }
  store_rows<T, DP, M>(o + ((long long)b * r.Tq * r.H + h) * r.D, (long long)r.H * r.D, acc, inv, q0, r.Tq, r.D, ty, tx);
}

// delta[b, h, t] = sum_d grad_out * (o + lo), a warp a row; o and lo (null: none) are contiguous.  Rows between Tq and `pitch` get zeros.
// 16-bit heads whose lanes have 16 bytes each are read as vectors.
template <typename T>
__global__ void __launch_bounds__(256) rules_delta_kernel(const T* o, const T* lo, const T* go, Strides gs, float* delta, int B, int H, int Tq, int pitch, int D, int vec) {
  const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= (long long)B * pitch * H) return;
  const int h = (int)(row % H), lane = threadIdx.x & 31;
  const long long bt = row / H;
  const int t = (int)(bt % pitch), b = (int)(bt / pitch);
  float sum = 0.f;
  if (t < Tq) {
    const long long at = (((long long)b * Tq + t) * H + h) * D;
    const T *x = o + at, *z = lo + at, *y = go + b * gs.b + t * gs.t + h * gs.h;
    if (vec) {
      constexpr int V = 16 / sizeof(T);
      for (int d = lane * V; d < D; d += 32 * V) {
        const uint4 a = *reinterpret_cast<const uint4*>(x + d), c = *reinterpret_cast<const uint4*>(y + d);
        const uint4 e = lo != nullptr ? *reinterpret_cast<const uint4*>(z + d) : make_uint4(0, 0, 0, 0);
        const T *xa = reinterpret_cast<const T*>(&a), *yc = reinterpret_cast<const T*>(&c), *ze = reinterpret_cast<const T*>(&e);
#pragma unroll
        for (int i = 0; i < V; ++i) sum = fmaf(to_f32<T>(xa[i]) + (lo != nullptr ? to_f32<T>(ze[i]) : 0.f), to_f32<T>(yc[i]), sum);
      }
    } else {
      for (int d = lane; d < D; d += 32) sum = fmaf(load_f32(x + d) + (lo != nullptr ? load_f32(z + d) : 0.f), load_f32(y + d), sum);
    }
    sum = warp_sum(sum);
  }
  if (lane == 0) delta[((long long)b * H + h) * pitch + t] = sum;
}

// The same where a row is G lanes of 16 bytes each: a group of lanes has four rows of one head, whose loads are all on their way before the first is
// used.  Bound by the bytes of the three tensors: 34 us at 2 x 4096 x 32 x 128 (5.9 TB/s), a warp a row 81 us.
template <typename T, int G>
__global__ void __launch_bounds__(256) rules_delta4_kernel(const T* o, const T* lo, const T* go, Strides gs, float* delta, int H, int Tq, int pitch, int D, long long n) {
  constexpr int V = 16 / sizeof(T), R = 4;
  const long long at = (long long)blockIdx.x * (256 / G) + threadIdx.x / G;
  const bool in = at < n;
  int h, t, b;
  if (n <= 0x7fffffffll) {
    const unsigned i = (unsigned)(in ? at : 0), bt = i / (unsigned)H;
    h = (int)(i % (unsigned)H);
    b = (int)(bt / (unsigned)(pitch / R));
    t = (int)(bt % (unsigned)(pitch / R)) * R;
  } else {
    const long long i = in ? at : 0, bt = i / H;
    h = (int)(i % H);
    b = (int)(bt / (pitch / R));
    t = (int)(bt % (pitch / R)) * R;
  }
  const int d = (threadIdx.x % G) * V;
  const bool mine = in && d < D;
  uint4 x[R], y[R], z[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    x[r] = y[r] = z[r] = make_uint4(0, 0, 0, 0);
    if (mine && t + r < Tq) {
      const long long from = (((long long)b * Tq + t + r) * H + h) * D + d;
      x[r] = *reinterpret_cast<const uint4*>(o + from);
      y[r] = *reinterpret_cast<const uint4*>(go + b * gs.b + (t + r) * gs.t + h * gs.h + d);
      if (lo != nullptr) z[r] = *reinterpret_cast<const uint4*>(lo + from);
    }
  }
  float sum[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    sum[r] = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float a = to_f32<T>(reinterpret_cast<const T*>(&x[r])[i]), c = to_f32<T>(reinterpret_cast<const T*>(&y[r])[i]);
      sum[r] = fmaf(a + to_f32<T>(reinterpret_cast<const T*>(&z[r])[i]), c, sum[r]);
    }
#pragma unroll
    for (int w = 1; w < G; w <<= 1) sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], w);
  }
  if (in && threadIdx.x % G == 0) *reinterpret_cast<float4*>(delta + ((long long)b * H + h) * pitch + t) = make_float4(sum[0], sum[1], sum[2], sum[3]);
}

template <typename T>
bool vectors(const void* p, const Strides& s, int D) {
  constexpr int V = 16 / sizeof(T);
  return D % V == 0 && s.t % V == 0 && s.h % V == 0 && s.b % V == 0 && ((uintptr_t)p & 15) == 0;
}

template <typename T>
void launch_delta(const T* o, const T* lo, const T* go, const Strides& os, const Strides& gs, float* delta, int B, int H, int Tq, int pitch, int D, cudaStream_t stream) {
  const bool vec = vectors<T>(o, os, D) && vectors<T>(lo, os, D) && vectors<T>(go, gs, D);
  const int lanes = D * (int)sizeof(T) / 16;
  const long long n = (long long)B * H * (pitch / 4);
  if (vec && lanes <= 32 && pitch % 4 == 0 && ((uintptr_t)delta & 15) == 0) {
#define KB_LANES(G) rules_delta4_kernel<T, G><<<(unsigned)((n + 256 / G - 1) / (256 / G)), 256, 0, stream>>>(o, lo, go, gs, delta, H, Tq, pitch, D, n)
    if (lanes <= 8) KB_LANES(8);
    else if (lanes <= 16) KB_LANES(16);
    else KB_LANES(32);
#undef KB_LANES
    return;
  }
  rules_delta_kernel<T><<<(unsigned)(((long long)B * pitch * H + 7) / 8), 256, 0, stream>>>(o, lo, go, gs, delta, B, H, Tq, pitch, D, vec);
}

// Probability of a pair and the gradient of its plain score, from the sums that the forward pass kept.
__device__ __forceinline__ void rule_gradient(const Rules& r, const Score& f, bool seen, float s, float dp, float lse, float delta, int i, int j, float& p, float& ds) {
  float through;
  const float x = rule_score(r, f, s, i, j, through);
  p = seen ? ex2(x - lse) : 0.f;
  ds = seen ? p * (dp - delta) * through : 0.f;
}

// A key tile's walk over the query heads of its group and their row tiles, and how many blocks share it.
struct Parts {
  int count;    // 1: gradients are stored as they are
  float* sums;  // [dk, dv][count][B, Tk, Hkv, D]
};
// dk and dv from the sums of their parts, in order.
template <typename T>
__global__ void __launch_bounds__(256) join_parts_kernel(const float* sums, T* dk, T* dv, int parts, long long n, float scale) {
  const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
  if (at >= 2 * n) return;
  const bool second = at >= n;
  const long long e = second ? at - n : at;
  const float* from = sums + (second ? (long long)parts * n : 0) + e;
  float x = from[0];
  for (int i = 1; i < parts; ++i) x += from[i * n];
  (second ? dv : dk)[e] = from_f32<T>(x * (second ? 1.f : scale));
}

template <typename T, int DP, int BT>
__global__ void __launch_bounds__(256) rules_dkv_kernel(const Rules r, const T* q, Strides qs, const T* k, Strides ks, const T* v, Strides vs, const Gradients g, T* dk, T* dv,
                                                        const Parts parts, int vec) {
  using C = Tile<T, DP, BT>;
  constexpr int M = BT / 16;
  extern __shared__ __align__(16) float sm[];
  float *sK = sm, *sV = sK + C::FLOATS, *sQ = sV + C::FLOATS, *sG = sQ + C::FLOATS, *sP = sG + C::FLOATS, *sD = sP + BT * C::SP, *sL = sD + BT * C::SP, *sE = sL + BT;
  int* sS = reinterpret_cast<int*>(sE + BT);
  const int unit = (int)(blockIdx.x / parts.count), part = (int)(blockIdx.x % parts.count);
  const int heads = r.Hkv * r.B, k0 = unit / heads * BT;  // a causal mask gives the first keys the most rows
  const int hkv = unit % heads % r.Hkv, b = unit % heads / r.Hkv, group = r.H / r.Hkv;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  load_tile<T, DP, BT>(sK, k + b * ks.b + hkv * ks.h, ks.t, k0, r.Tk, r.D, vec & 2);
  load_tile<T, DP, BT>(sV, v + b * vs.b + hkv * vs.h, vs.t, k0, r.Tk, r.D, vec & 4);
  const int prefix = prefix_of(r, b);
  float ak[M][DP / 16], av[M][DP / 16];
  int seg_k[M];
#pragma unroll
  for (int i = 0; i < M; ++i) {
    seg_k[i] = r.seg_k != nullptr && k0 + ty + 16 * i < r.Tk ? r.seg_k[(long long)b * r.Tk + k0 + ty + 16 * i] : 0;
#pragma unroll
    for (int e = 0; e < DP / 16; ++e) ak[i][e] = av[i][e] = 0.f;
  }
  int first, last;
  rows_of_keys(r, k0, min(k0 + BT, r.Tk) - 1, prefix, first, last);
  // the walk over the group's heads and their tiles of rows, or a part of it
  const int tiles = last >= first ? last / BT - first / BT + 1 : 0;
  const long long total = (long long)tiles * group, per = (total + parts.count - 1) / parts.count, begin = part * per, end = begin + per < total ? begin + per : total;
  for (int h = hkv * group + (tiles > 0 ? (int)(begin / tiles) : 0); h < (hkv + 1) * group; ++h) {
    const long long at = (long long)(h - hkv * group) * tiles;  // of the head's first tile
    if (at >= end) break;
    const Score f = score_of(r, h);
    const float *lse = g.lse + ((long long)b * r.H + h) * g.pitch, *delta = g.delta + ((long long)b * r.H + h) * g.pitch;
    const int from = (int)(begin > at ? begin - at : 0), to = (int)(end - at < tiles ? end - at : tiles);
    for (int n = from; n < to; ++n) {
      const int q0 = (first / BT + n) * BT;
      if (!segments_meet(r, b, q0, k0)) continue;
      __syncthreads();
      load_tile<T, DP, BT>(sQ, q + b * qs.b + h * qs.h, qs.t, q0, r.Tq, r.D, vec & 1);
      load_tile<T, DP, BT>(sG, (const T*)g.grad_out + b * g.go.b + h * g.go.h, g.go.t, q0, r.Tq, r.D, vec & 8);
      for (int e = threadIdx.x; e < BT; e += 256) {
        const bool in = q0 + e < r.Tq;
        sL[e] = in ? lse[q0 + e] : INFINITY;
        sE[e] = in ? delta[q0 + e] : 0.f;
        sS[e] = r.seg_q != nullptr && in ? r.seg_q[(long long)b * r.Tq + q0 + e] : 0;
      }
      __syncthreads();
      float s[M][M], dp[M][M];
      product_rows<DP, M, C::PITCH>(s, sK, sQ, ty, tx);
      product_rows<DP, M, C::PITCH>(dp, sV, sG, ty, tx);
#pragma unroll
      for (int j = 0; j < M; ++j) {
        const int c = tx + 16 * j, t = q0 + c;
        int lo, hi;
        row_span(r, t, prefix, lo, hi);
        const int seg = sS[c];
#pragma unroll
        for (int i = 0; i < M; ++i) {
          const int key = k0 + ty + 16 * i;
          const bool seen = t < r.Tq && key >= lo && key <= hi && (r.seg_q == nullptr || (seg >= 0 && seg == seg_k[i]));
          float p, ds;
          rule_gradient(r, f, seen, s[i][j], dp[i][j], sL[c], sE[c], t, key, p, ds);
          sP[(ty + 16 * i) * C::SP + c] = p;
          sD[(ty + 16 * i) * C::SP + c] = ds;
        }
      }
      __syncwarp();
      product_cols<DP, BT, M, C::PITCH, C::SP>(av, sP, sG, ty, tx);
      product_cols<DP, BT, M, C::PITCH, C::SP>(ak, sD, sQ, ty, tx);
    }
  }
  float one[M], scale[M];
#pragma unroll
  for (int i = 0; i < M; ++i) {
    one[i] = 1.f;
    scale[i] = r.scale;
  }
  const long long base = ((long long)b * r.Tk * r.Hkv + hkv) * r.D, pitch = (long long)r.Hkv * r.D;
  if (parts.count > 1) {
    const long long size = (long long)r.B * r.Tk * r.Hkv * r.D;
    store_rows<float, DP, M>(parts.sums + part * size + base, pitch, ak, one, k0, r.Tk, r.D, ty, tx);
    store_rows<float, DP, M>(parts.sums + (parts.count + part) * size + base, pitch, av, one, k0, r.Tk, r.D, ty, tx);
    return;
  }
  store_rows<T, DP, M>(dk + base, pitch, ak, scale, k0, r.Tk, r.D, ty, tx);
  store_rows<T, DP, M>(dv + base, pitch, av, one, k0, r.Tk, r.D, ty, tx);
}

template <typename T, int DP, int BT>
__global__ void __launch_bounds__(256) rules_dq_kernel(const Rules r, const T* q, Strides qs, const T* k, Strides ks, const T* v, Strides vs, const Gradients g, T* dq, int vec) {
  using C = Tile<T, DP, BT>;
  constexpr int M = BT / 16;
  extern __shared__ __align__(16) float sm[];
  float *sQ = sm, *sG = sQ + C::FLOATS, *sK = sG + C::FLOATS, *sV = sK + C::FLOATS, *sD = sV + C::FLOATS;
  const int heads = r.H * r.B, n_q = (r.Tq + BT - 1) / BT;
  const int q0 = (n_q - 1 - (int)(blockIdx.x / heads)) * BT;
  const int h = (int)(blockIdx.x % heads) % r.H, b = (int)(blockIdx.x % heads) / r.H, hkv = h / (r.H / r.Hkv);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  load_tile<T, DP, BT>(sQ, q + b * qs.b + h * qs.h, qs.t, q0, r.Tq, r.D, vec & 1);
  load_tile<T, DP, BT>(sG, (const T*)g.grad_out + b * g.go.b + h * g.go.h, g.go.t, q0, r.Tq, r.D, vec & 8);
  const Score f = score_of(r, h);
  const int prefix = prefix_of(r, b);
  int lo[M], hi[M], seg[M], first, last;
  float lse[M], delta[M], acc[M][DP / 16], scale[M];
  keys_of_rows(r, q0, min(q0 + BT, r.Tq) - 1, prefix, first, last);
#pragma unroll
  for (int i = 0; i < M; ++i) {
    const int t = q0 + ty + 16 * i;
    const long long at = ((long long)b * r.H + h) * g.pitch + t;
    row_span(r, t, prefix, lo[i], hi[i]);
    seg[i] = r.seg_q != nullptr && t < r.Tq ? r.seg_q[(long long)b * r.Tq + t] : 0;
    if (t >= r.Tq || seg[i] < 0) hi[i] = -1;
    lse[i] = t < r.Tq ? g.lse[at] : INFINITY;
    delta[i] = t < r.Tq ? g.delta[at] : 0.f;
    scale[i] = r.scale;
#pragma unroll
    for (int e = 0; e < DP / 16; ++e) acc[i][e] = 0.f;
  }
  for (int k0 = first / BT * BT; k0 <= last; k0 += BT) {
    if (!segments_meet(r, b, q0, k0)) continue;
    __syncthreads();
    load_tile<T, DP, BT>(sK, k + b * ks.b + hkv * ks.h, ks.t, k0, r.Tk, r.D, vec & 2);
    load_tile<T, DP, BT>(sV, v + b * vs.b + hkv * vs.h, vs.t, k0, r.Tk, r.D, vec & 4);
    __syncthreads();
    float s[M][M], dp[M][M];
    product_rows<DP, M, C::PITCH>(s, sQ, sK, ty, tx);
    product_rows<DP, M, C::PITCH>(dp, sG, sV, ty, tx);
#pragma unroll
    for (int j = 0; j < M; ++j) {
      const int c = tx + 16 * j, key = k0 + c;
      const int seg_k = r.seg_k != nullptr && key < r.Tk ? r.seg_k[(long long)b * r.Tk + key] : 0;
#pragma unroll
      for (int i = 0; i < M; ++i) {
        const bool seen = key >= lo[i] && key <= hi[i] && (r.seg_k == nullptr || seg_k == seg[i]);
        float p, ds;
        rule_gradient(r, f, seen, s[i][j], dp[i][j], lse[i], delta[i], q0 + ty + 16 * i, key, p, ds);
        sD[(ty + 16 * i) * C::SP + c] = ds;
      }
    }
    __syncwarp();
    product_cols<DP, BT, M, C::PITCH, C::SP>(acc, sD, sK, ty, tx);
  }
  store_rows<T, DP, M>(dq + ((long long)b * r.Tq * r.H + h) * r.D, (long long)r.H * r.D, acc, scale, q0, r.Tq, r.D, ty, tx);
}

// Lowest and highest id that is not negative, and whether there is a negative one, of every SEG_TILE positions: a warp each.
__global__ void __launch_bounds__(128) segment_ranges_kernel(const int* seg, int4* out, int T, long long n) {
  const long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (w >= n) return;
  const int tiles = n_ranges(T), lane = threadIdx.x & 31, t0 = (int)(w % tiles) * SEG_TILE;
  const int* row = seg + w / tiles * T;
  int lo = INT_MAX, hi = -1, none = 0;
#pragma unroll
  for (int i = 0; i < SEG_TILE / 32; ++i) {
    const int t = t0 + i * 32 + lane;
    if (t < T) {
      const int s = row[t];
      if (s < 0) none = 1;
      else {
        lo = min(lo, s);
        hi = max(hi, s);
      }
    }
  }
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  none = __any_sync(0xffffffffu, none);
  if (lane == 0) out[w] = make_int4(lo, hi, none, 0);
}

template <typename T, int DP, int BT>
int rules_fwd(const Rules& r, const void* q, Strides qs, const void* k, Strides ks, const void* v, Strides vs, void* o, float* lse, int pitch, cudaStream_t stream) {
  using C = Tile<T, DP, BT>;
  constexpr int SMEM = (3 * C::FLOATS + BT * C::SP) * 4;
  static bool attr[KB_MAX_DEVICES] = {false};
  if (!kb_allow_smem(rules_fwd_kernel<T, DP, BT>, SMEM, attr)) {
    kb200_set_error("attention_rules: shared-memory limit");
    return -3;
  }
  const int vec = (vectors<T>(q, qs, r.D) ? 1 : 0) | (vectors<T>(k, ks, r.D) ? 2 : 0) | (vectors<T>(v, vs, r.D) ? 4 : 0);
  rules_fwd_kernel<T, DP, BT><<<(unsigned)((long long)((r.Tq + BT - 1) / BT) * r.H * r.B), 256, SMEM, stream>>>(r, (const T*)q, qs, (const T*)k, ks, (const T*)v, vs, (T*)o, lse, pitch, vec);
  return 0;
}
template <typename T, int DP, int BT>
int rules_bwd(const Rules& r, const void* q, Strides qs, const void* k, Strides ks, const void* v, Strides vs, const Gradients& g, void* dq, void* dk, void* dv,
              const Parts& parts, cudaStream_t stream) {
  using C = Tile<T, DP, BT>;
  constexpr int SMEM_KV = (4 * C::FLOATS + 2 * BT * C::SP + 3 * BT) * 4, SMEM_Q = (4 * C::FLOATS + BT * C::SP) * 4;
  static bool attr[2][KB_MAX_DEVICES] = {{false}};
  if (!kb_allow_smem(rules_dkv_kernel<T, DP, BT>, SMEM_KV, attr[0]) || !kb_allow_smem(rules_dq_kernel<T, DP, BT>, SMEM_Q, attr[1])) {
    kb200_set_error("attention_rules: shared-memory limit");
    return -3;
  }
  const int vec = (vectors<T>(q, qs, r.D) ? 1 : 0) | (vectors<T>(k, ks, r.D) ? 2 : 0) | (vectors<T>(v, vs, r.D) ? 4 : 0) | (vectors<T>(g.grad_out, g.go, r.D) ? 8 : 0);
  if (dk != nullptr)
    rules_dkv_kernel<T, DP, BT><<<(unsigned)((long long)((r.Tk + BT - 1) / BT) * r.Hkv * r.B * parts.count), 256, SMEM_KV, stream>>>(r, (const T*)q, qs, (const T*)k, ks, (const T*)v, vs, g,
                                                                                                                   (T*)dk, (T*)dv, parts, vec);
  if (dk != nullptr && parts.count > 1) {
    const long long n = (long long)r.B * r.Tk * r.Hkv * r.D;
    join_parts_kernel<T><<<(unsigned)((2 * n + 255) / 256), 256, 0, stream>>>(parts.sums, (T*)dk, (T*)dv, parts.count, n, r.scale);
  }
  if (dq != nullptr)
    rules_dq_kernel<T, DP, BT><<<(unsigned)((long long)((r.Tq + BT - 1) / BT) * r.H * r.B), 256, SMEM_Q, stream>>>(r, (const T*)q, qs, (const T*)k, ks, (const T*)v, vs, g, (T*)dq, vec);
  return 0;
}

}  // namespace

// Ids [B, T] of segments to their ranges, [B, ceil(T / 128)] of four ints each.
KB_API int kb200_segment_ranges(const int* seg, void* ranges, int B, int T, cudaStream_t stream) {
  const long long n = (long long)B * ((T + SEG_TILE - 1) / SEG_TILE);
  if (n <= 0) return 0;
  segment_ranges_kernel<<<(unsigned)((n + 3) / 4), 128, 0, stream>>>(seg, (int4*)ranges, T, n);
  KB_CHECK_LAUNCH("segment_ranges");
  return 0;
}

namespace {
bool check(const Rules& r, int dtype) {
  if (r.B <= 0 || r.H <= 0 || r.Hkv <= 0 || r.H % r.Hkv || r.Tq <= 0 || r.Tk <= 0 || r.D <= 0 || r.D > 256 || dtype < 0 || dtype > 2) {
    kb200_set_error("attention_rules: sizes out of range (heads of up to 256, query heads a multiple of key heads)");
    return false;
  }
  if (r.Tq > (1 << 30) || r.Tk > (1 << 30) || ((long long)((r.Tq + 31) / 32) * r.H * r.B) > 0x7fffffffll || ((long long)((r.Tk + 31) / 32) * r.H * r.B) > 0x7fffffffll) {
    kb200_set_error("attention_rules: too many rows");
    return false;
  }
  return true;
}
}  // namespace

#define KB_RULES_DISPATCH(CALL)                                       \
  do {                                                                \
    if (r.D <= 64) {                                                  \
      if (dtype == 0) rc = CALL(float, 64, 64);                       \
      else if (dtype == 1) rc = CALL(__nv_bfloat16, 64, 64);          \
      else rc = CALL(__half, 64, 64);                                 \
    } else if (r.D <= 128) {                                          \
      if (dtype == 0) rc = CALL(float, 128, 64);                      \
      else if (dtype == 1) rc = CALL(__nv_bfloat16, 128, 64);         \
      else rc = CALL(__half, 128, 64);                                \
    } else {                                                          \
      if (dtype == 0) rc = CALL(float, 256, 32);                      \
      else if (dtype == 1) rc = CALL(__nv_bfloat16, 256, 32);         \
      else rc = CALL(__half, 256, 32);                                \
    }                                                                 \
  } while (0)

// q [B, Tq, H, D], k and v [B, Tk, Hkv, D] with unit stride on D; o [B, Tq, H, D] contiguous; lse [B, H, pitch] (log2 units; +inf: a row that
// sees nothing) may be null.  dtype 0 float32, 1 bfloat16, 2 float16.
KB_API int kb200_attention_rules_fwd(const void* q, const void* k, const void* v, void* o, float* lse, int pitch, const long long* strides, int dtype, int B, int H, int Hkv, int Tq,
                                     int Tk, int D, float scale, float cap, const float* slopes, int causal, int window, const int* prefix, const int* seg_q, const int* seg_k,
                                     const void* range_q, const void* range_k, cudaStream_t stream) {
  const Rules r{B, H, Hkv, Tq, Tk, D, scale, cap, slopes, causal, window, prefix, seg_q, seg_k, (const int4*)range_q, (const int4*)range_k};
  if (!check(r, dtype)) return -2;
  const Strides qs{strides[0], strides[1], strides[2]}, ks{strides[3], strides[4], strides[5]}, vs{strides[6], strides[7], strides[8]};
  int rc = 0;
#define KB_CALL(T, DP, BT) rules_fwd<T, DP, BT>(r, q, qs, k, ks, v, vs, o, lse, pitch, stream)
  KB_RULES_DISPATCH(KB_CALL);
#undef KB_CALL
  if (rc != 0) return rc;
  KB_CHECK_LAUNCH("attention_rules_fwd");
  return 0;
}

// delta [B, H, pitch]: for each row the sum of grad_out * (o + lo); lo may be null.
KB_API int kb200_attention_rules_delta(const void* o, const void* lo, const void* grad_out, const long long* strides, float* delta, int pitch, int dtype, int B, int H, int Tq, int D,
                                       cudaStream_t stream) {
  const Strides gs{strides[0], strides[1], strides[2]};
  const long long blocks = ((long long)B * pitch * H + 7) / 8;
  if (pitch < Tq || blocks > 0x7fffffffll || dtype < 0 || dtype > 2) {
    kb200_set_error("attention_rules_delta: sizes out of range");
    return -2;
  }
  const Strides os{(long long)H * D, D, (long long)Tq * H * D};
#define KB_DELTA(T) launch_delta<T>((const T*)o, (const T*)lo, (const T*)grad_out, os, gs, delta, B, H, Tq, pitch, D, stream)
  if (dtype == 0) KB_DELTA(float);
  else if (dtype == 1) KB_DELTA(__nv_bfloat16);
  else KB_DELTA(__half);
#undef KB_DELTA
  KB_CHECK_LAUNCH("attention_rules_delta");
  return 0;
}

namespace {
// Parts of a key tile's walk: with fewer key tiles than two blocks an SM, as many as make up two, of two tiles of rows each at least.
int parts_of(int B, int H, int Hkv, int Tq, int Tk, int D) {
  const long long BT = D <= 128 ? 64 : 32, units = (Tk + BT - 1) / BT * Hkv * B, blocks = 2ll * kb_sm_count(), walk = (long long)(H / Hkv) * ((Tq + BT - 1) / BT);
  if (units >= blocks) return 1;
  const long long want = (blocks + units - 1) / units, most = walk / 2 < 16 ? walk / 2 : 16;
  return (int)(want < most ? want : most > 1 ? most : 1);
}
}  // namespace

// Floats of workspace that kb200_attention_rules_bwd takes for dk and dv at these sizes.
KB_API long long kb200_attention_rules_bwd_work_plain(int B, int H, int Hkv, int Tq, int Tk, int D) {
  if (B <= 0 || Hkv <= 0 || H < Hkv || Tq <= 0 || Tk <= 0 || D <= 0) return 0;
  const int parts = parts_of(B, H, Hkv, Tq, Tk, D);
  return parts > 1 ? 2ll * parts * B * Tk * Hkv * D : 0;
}

// Gradients of the above: dq [B, Tq, H, D], dk and dv [B, Tk, Hkv, D] contiguous; dq, or dk and dv together, may be null.  work: `floats` of them, as many as
// kb200_attention_rules_bwd_work_plain says, or null.
KB_API int kb200_attention_rules_bwd(const void* q, const void* k, const void* v, const void* grad_out, const long long* strides, const float* lse, const float* delta, int pitch,
                                     void* dq, void* dk, void* dv, int dtype, int B, int H, int Hkv, int Tq, int Tk, int D, float* work, long long floats, float scale, float cap, const float* slopes, int causal, int window,
                                     const int* prefix, const int* seg_q, const int* seg_k, const void* range_q, const void* range_k, cudaStream_t stream) {
  const Rules r{B, H, Hkv, Tq, Tk, D, scale, cap, slopes, causal, window, prefix, seg_q, seg_k, (const int4*)range_q, (const int4*)range_k};
  if (!check(r, dtype)) return -2;
  const Strides qs{strides[0], strides[1], strides[2]}, ks{strides[3], strides[4], strides[5]}, vs{strides[6], strides[7], strides[8]};
  const Gradients g{grad_out, {strides[9], strides[10], strides[11]}, lse, delta, pitch};
  Parts parts{parts_of(B, H, Hkv, Tq, Tk, D), work};
  if (work == nullptr || 2ll * parts.count * B * Tk * Hkv * D > floats) parts.count = 1;
  int rc = 0;
#define KB_CALL(T, DP, BT) rules_bwd<T, DP, BT>(r, q, qs, k, ks, v, vs, g, dq, dk, dv, parts, stream)
  KB_RULES_DISPATCH(KB_CALL);
#undef KB_CALL
  if (rc != 0) return rc;
  KB_CHECK_LAUNCH("attention_rules_bwd");
  return 0;
}

// All of a gradient in one call: delta, from o, lo (may be null) and grad_out, then the above.  err is unused.
KB_API int kb200_attention_rules_grads(const void* q, const void* k, const void* v, const void* o, const void* lo, const void* grad_out, const long long* strides, const float* lse,
                                       float* delta, int pitch, void* dq, void* dk, void* dv, int dtype, int B, int H, int Hkv, int Tq, int Tk, int D, int* err, float* work, long long floats, float scale, float cap,
                                       const float* slopes, int causal, int window, const int* prefix, const int* seg_q, const int* seg_k, const void* range_q, const void* range_k,
                                       cudaStream_t stream) {
  (void)err;
  const int rc = kb200_attention_rules_delta(o, lo, grad_out, strides + 9, delta, pitch, dtype, B, H, Tq, D, stream);
  return rc != 0 ? rc
                 : kb200_attention_rules_bwd(q, k, v, grad_out, strides, lse, delta, pitch, dq, dk, dv, dtype, B, H, Hkv, Tq, Tk, D, work, floats, scale, cap, slopes, causal, window, prefix, seg_q,
                                             seg_k, range_q, range_k, stream);
}
