// Attention of new tokens over a paged key/value cache, with their keys and values added to it in the same launch.
//
// The cache is two pools of pages, [P, page, Hkv, D] each; pages[b, n] names the pool's page that holds positions n * page .. of sequence b.
// A call brings T new tokens a sequence.  Their keys and values go to positions n .. n + T - 1 (n = lengths[b]), and the query of token t
// sees the positions up to n + t, within the window if there is one.  Scores are those of attention_rules.cuh: cap and slopes.
//
// A decoder's step reads each key and value once and does little else, so the cache's bytes bound it.  One sequence and key head is the
// work of a thread-block cluster: its CTAs take equal parts of the visible positions, each with a running maximum and sum, and join
// their parts through distributed shared memory: one launch, no workspace, and the same order of sums every time.  Few long sequences are split
// into more parts than a cluster has, one wave over the chip, which leave their sums in a workspace for a second launch.  The T * H / Hkv rows
// that share a key head share its loads.
//
// A negative length marks an idle sequence: nothing is written and its rows are zero.  A position whose page is missing (behind the end of
// the table, or outside of the pool) is neither read nor written; rows that would have seen it are NaN.
#include <cooperative_groups.h>

#include "attention_rules.cuh"

namespace {
using namespace kbrules;
namespace cg = cooperative_groups;

struct Cache {
  int B, H, Hkv, T, D, n_pages, page, wide;  // pages in the pool, positions a page, pages a sequence
  long long pool_p, pool_t, pool_h;          // strides of the pools in elements
  Strides q, k, v;                           // of the new tokens; the output is contiguous
  const int *pages, *lengths;
  float scale, cap;
  const float* slopes;
  int window;
};

constexpr int KEYS = 32;   // a tile
constexpr int ROWS = 16;   // rows of a block at most
constexpr int THREADS = 128;

template <int DP>
struct CacheTile {
  static constexpr int PITCH = DP + 4;
  static constexpr int FLOATS = ROWS * PITCH + KEYS * PITCH * 2 + ROWS * (KEYS + 1) + 3 * ROWS;
};

// Parts that do not join within a cluster leave their rows, maxima and sums here; join_kernel adds them up.
struct Parts {
  float* rows;  // [units][parts][rows of a unit][D], null: join in the cluster
  float2* sums; // [units][parts][rows of a unit]: maximum, sum
  int count;
};

template <typename T, int DP>
__global__ void __launch_bounds__(THREADS) cache_kernel(const Cache c, const T* q, const T* new_k, const T* new_v, T* pool_k, T* pool_v, T* out, const Parts ws, int vec) {
  constexpr int PITCH = CacheTile<DP>::PITCH, COLS = DP / THREADS > 0 ? DP / THREADS : 1;
  extern __shared__ __align__(16) float sm[];
  float *sQ = sm, *sK = sQ + ROWS * PITCH, *sV = sK + KEYS * PITCH, *sP = sV + KEYS * PITCH, *sM = sP + ROWS * (KEYS + 1), *sL = sM + ROWS, *sA = sL + ROWS;
  __shared__ int s_bad[KEYS];
  cg::cluster_group cluster = cg::this_cluster();
  const bool joined = ws.rows == nullptr;
  const int parts = joined ? (int)cluster.num_blocks() : ws.count, part = (int)(blockIdx.x % parts);
  const int G = c.H / c.Hkv, rows = c.T * G, row_tiles = (rows + ROWS - 1) / ROWS;
  const int unit = (int)(blockIdx.x / parts), rt = unit % row_tiles, hkv = unit / row_tiles % c.Hkv, b = unit / row_tiles / c.Hkv;
  const int r0 = rt * ROWS, nr = min(ROWS, rows - r0);  // row r: token r / G, query head hkv * G + r % G
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const long long n = c.lengths[b];
  const long long last = n < 0 ? -1 : n + (r0 + nr - 1) / G;  // of the positions that any row sees
  // a length behind the table's end: every row sees its own position, which has no page, and is NaN, whatever there is before
  const long long first = n < 0 ? 0 : n >= (long long)c.wide * c.page ? n + r0 / G : c.window > 0 ? max(0ll, n + r0 / G - c.window + 1) : 0;
  // parts of whole tiles
  const long long tiles = (last - first + KEYS) / KEYS, per = (tiles + parts - 1) / parts;
  const long long from = first + part * per * KEYS, to = min(last, from + per * KEYS - 1);

  for (int e = tid; e < ROWS * DP; e += THREADS) {
    const int r = e / DP, d = e % DP, t = (r0 + r) / G, h = hkv * G + (r0 + r) % G;
    sQ[r * PITCH + d] = r < nr && d < c.D ? load_f32(q + b * c.q.b + t * c.q.t + h * c.q.h + d) : 0.f;
  }
  if (tid < ROWS) {
    sM[tid] = -INFINITY;
    sL[tid] = 0.f;
  }
  float acc[ROWS][COLS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r)
#pragma unroll
    for (int e = 0; e < COLS; ++e) acc[r][e] = 0.f;

  for (long long k0 = from; k0 <= to; k0 += KEYS) {
    __syncthreads();
    if (tid < KEYS) {
      const long long pos = k0 + tid, slot = pos / c.page;
      s_bad[tid] = 0;
      if (pos <= to) {
        const int p = slot < c.wide ? c.pages[(long long)b * c.wide + slot] : -1;
        s_bad[tid] = p < 0 || p >= c.n_pages ? -1 : p + 1;
      }
    }
    __syncthreads();
    // keys and values as float32, new ones from the call (and into their page), zeros where there is none
    constexpr int V = 16 / sizeof(T);
    const int step = vec ? V : 1, per_row = DP / step;
    for (int e = tid; e < KEYS * per_row; e += THREADS) {
      const int i = e / per_row, d = (e % per_row) * step;
      const long long pos = k0 + i;
      const int p = s_bad[i];
      const bool in = pos <= to && d < c.D, fresh = in && pos >= n;
      const long long at = p > 0 ? (long long)(p - 1) * c.pool_p + (pos % c.page) * c.pool_t + hkv * c.pool_h + d : 0;
      const T *ks = pool_k + at, *vs = pool_v + at;
      if (fresh) {
        ks = new_k + b * c.k.b + (pos - n) * c.k.t + hkv * c.k.h + d;
        vs = new_v + b * c.v.b + (pos - n) * c.v.t + hkv * c.v.h + d;
      }
      // a token is added by the CTA that has its first row: that row sees it, whatever the window
      const long long own_row = (pos - n) * G;
      const bool read = in && (fresh || p > 0), keep = fresh && p > 0 && own_row >= r0 && own_row < r0 + nr;
      if (vec) {
        uint4 x = make_uint4(0, 0, 0, 0), y = x;
        if (read) {
          x = *reinterpret_cast<const uint4*>(ks);
          y = *reinterpret_cast<const uint4*>(vs);
        }
        if (keep) {
          *reinterpret_cast<uint4*>(pool_k + at) = x;
          *reinterpret_cast<uint4*>(pool_v + at) = y;
        }
        const T *xt = reinterpret_cast<const T*>(&x), *yt = reinterpret_cast<const T*>(&y);
#pragma unroll
        for (int u = 0; u < V; ++u) {
          sK[i * PITCH + d + u] = to_f32<T>(xt[u]);
          sV[i * PITCH + d + u] = to_f32<T>(yt[u]);
        }
      } else {
        const T x = read ? *ks : from_f32<T>(0.f), y = read ? *vs : from_f32<T>(0.f);
        if (keep) {
          pool_k[at] = x;
          pool_v[at] = y;
        }
        sK[i * PITCH + d] = to_f32<T>(x);
        sV[i * PITCH + d] = to_f32<T>(y);
      }
    }
    __syncthreads();
    // a lane a key, a warp every fourth row
    for (int r = warp; r < nr; r += 4) {
      const int t = (r0 + r) / G, h = hkv * G + (r0 + r) % G;
      const long long pos = k0 + lane, back = n + t - pos;
      float s = 0.f;
#pragma unroll 8
      for (int d = 0; d < DP; d += 4) {
        const float4 x = *reinterpret_cast<const float4*>(sQ + r * PITCH + d), y = *reinterpret_cast<const float4*>(sK + lane * PITCH + d);
        s = fmaf(x.x, y.x, fmaf(x.y, y.y, fmaf(x.z, y.z, fmaf(x.w, y.w, s))));
      }
      float x = s * (c.scale * LOG2E);
      if (c.cap > 0.f) x = tanh_any(s * (c.scale / c.cap)) * (c.cap * LOG2E);
      if (c.slopes != nullptr) x = fmaf(-c.slopes[h] * LOG2E, (float)back, x);
      if (s_bad[lane] < 0) x = NAN;
      if (pos > to || back < 0 || (c.window > 0 && back >= c.window)) x = -INFINITY;
      const bool bad = __any_sync(0xffffffffu, x != x);
      const float m = sM[r], m_new = fmaxf(m, warp_max(x)), base = m_new == -INFINITY ? 0.f : m_new;
      const float p = bad ? NAN : ex2(x - base), alpha = ex2(m - base), sum = warp_sum(p);
      sP[r * (KEYS + 1) + lane] = p;
      __syncwarp();
      if (lane == 0) {
        sM[r] = m_new;
        sL[r] = fmaf(sL[r], alpha, sum);
        sA[r] = alpha;
      }
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < COLS; ++e) {
      const int d = tid + e * THREADS;
      if (d < DP) {
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
          if (r < nr) acc[r][e] *= sA[r];
        for (int i = 0; i < KEYS; ++i) {
          const float y = sV[i * PITCH + d];
#pragma unroll
          for (int r = 0; r < ROWS; ++r)
            if (r < nr) acc[r][e] = fmaf(sP[r * (KEYS + 1) + i], y, acc[r][e]);
        }
      }
    }
  }
  __syncthreads();
  if (!joined) {
    const long long at = ((long long)unit * parts + part) * ROWS;
#pragma unroll
    for (int e = 0; e < COLS; ++e) {
      const int d = tid + e * THREADS;
      if (d < DP)
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
          if (r < nr) ws.rows[(at + r) * DP + d] = acc[r][e];
    }
    if (tid < ROWS) ws.sums[at + tid] = make_float2(sM[tid], sL[tid]);
    return;
  }
  // this CTA's part over its query tile: [row][column]
#pragma unroll
  for (int e = 0; e < COLS; ++e) {
    const int d = tid + e * THREADS;
    if (d < DP)
#pragma unroll
      for (int r = 0; r < ROWS; ++r) sQ[r * PITCH + d] = acc[r][e];
  }
  cluster.sync();
  for (int r = part; r < nr; r += parts) {
    float m = -INFINITY, l = 0.f;
    for (int i = 0; i < parts; ++i) m = fmaxf(m, cluster.map_shared_rank(sM, i)[r]);
    const float base = m == -INFINITY ? 0.f : m;
    for (int i = 0; i < parts; ++i) l = fmaf(cluster.map_shared_rank(sL, i)[r], ex2(cluster.map_shared_rank(sM, i)[r] - base), l);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int t = (r0 + r) / G, h = hkv * G + (r0 + r) % G;
    for (int d = tid; d < c.D; d += THREADS) {
      float x = 0.f;
      for (int i = 0; i < parts; ++i) x = fmaf(cluster.map_shared_rank(sQ, i)[r * PITCH + d], ex2(cluster.map_shared_rank(sM, i)[r] - base), x);
      out[(((long long)b * c.T + t) * c.H + h) * c.D + d] = from_f32<T>(x * inv);
    }
  }
  cluster.sync();  // nobody leaves while its part is read
}

// ------------------------------------------------------------------------------------------------ 16-bit heads of up to 128
// Every warp works by itself, on tiles of 16 positions in turn, and keeps them in registers: the products (mma.sync: a step has few rows, and the
// bytes bound it) take the positions, or the columns, as their 16 rows and the queries' rows as their 8 columns.
//   S^T = K Q^T   a lane (g = lane / 4, t = lane % 4) holds 16 bytes of keys g and g + 8 at a time: eight columns, the operand of two steps.  Which
//                 columns make up a step does not matter as long as Q is read the same way.
//   O^T = V^T P^T a lane holds 16 bytes of the values 2t, 2t + 1, 2t + 8, 2t + 9 and pairs them up; P^T is S^T's own layout transposed (movmatrix).
// So keys and values go from memory to the products without shared memory in between, and while one tile is worked on the loads of the next
// are on their way: 8 KB a warp, 96 KB an SM.  Where a tile lies in one page its address is the same for the whole warp.  No barrier until
// the warps, and then the cluster's blocks, join their parts.
// Measured, of 6542 GB/s: two sequences of 65000 positions, 8 key heads of 128, 91 us (5.85 TB/s); 64 of 200 to 4000 122 us (4.4 TB/s: blocks of unequal
// length in 2.3 waves); 16 of which a window leaves 1024, 5 tokens each, 40 us (3.3 TB/s: 256 blocks on 148 SMs); one of 900 7.2 us, a chain of waits for
// memory.  With float32 in shared memory and the FMA pipes these took 3037, 1534, 261 and 12 us.
constexpr int TILE_16 = 16;

template <typename T>
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma<__nv_bfloat16>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma<__half>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pair16(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pair16(float a, float b, __half) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ uint4 load_once(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// What a position that is not there, and a column beyond the head's size, reads: an address is chosen, never a value after its load, or the load
// would be waited for on the spot.
__device__ uint4 zero_row[16];  // as long as the widest head

// tanh(x * pre) * post of a lane's four scores, for a warp: the polynomial of tanh_small2's kind where no lane has a value beyond 1/2
__device__ __forceinline__ void capped4(float (&x)[4], float pre, float post) {
  float top = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[e] *= pre;
    top = fmaxf(top, fabsf(x[e]));
  }
  if (!__any_sync(0xffffffffu, top > 0.5f)) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {  // x times a polynomial of degree 3 in x^2, fitted on [-1/2, 1/2]: 5.5e-7 of the value
      const float u = x[e] * x[e];
      x[e] *= fmaf(fmaf(fmaf(-0.04440227895975113f, u, 0.13190299272537231f), u, -0.33326318860054016f), u, 0.999999463558197f) * post;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = tanh_any(x[e]) * post;
  }
}

// NT: eights of rows that a block works on; FULL: the head's size is DP.  Four warps, two or three blocks an SM: one's end hides behind another's middle.
template <typename T, int DP, int NT, bool FULL>
__global__ void __launch_bounds__(128, NT == 1 ? 3 : 2) cache_kernel_16(const Cache c, const T* q, const T* new_k, const T* new_v, T* pool_k, T* pool_v, T* out, const Parts ws) {
  constexpr int W = 4, ROWS_ = 8 * NT, CH = DP / 32, VH = DP / 64, MT = DP / 16;  // 16-byte chunks of a key and of a value a lane; tiles of 16 columns
  constexpr int PITCH = DP + 4;
  __shared__ float s_own[W * ROWS_ * PITCH], s_part[ROWS_ * PITCH], s_m[W * ROWS_], s_l[W * ROWS_], s_f[W * ROWS_];
  cg::cluster_group cluster = cg::this_cluster();
  const bool joined = ws.rows == nullptr;
  const int parts = joined ? (int)cluster.num_blocks() : ws.count, part = (int)(blockIdx.x % parts);
  const int G = c.H / c.Hkv, rows = c.T * G, row_tiles = (rows + ROWS_ - 1) / ROWS_;
  const int unit = (int)(blockIdx.x / parts), rt = unit % row_tiles, hkv = unit / row_tiles % c.Hkv, b = unit / row_tiles / c.Hkv;
  const int r0 = rt * ROWS_, nr = min(ROWS_, rows - r0);  // row r: token r / G, query head hkv * G + r % G
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  const int length = c.lengths[b];
  const uint32_t n = length < 0 ? 0u : (uint32_t)length;  // positions fit 32 bits without a sign: T is at most 2^30
  const bool idle = length < 0;
  const uint32_t last = n + (uint32_t)((r0 + nr - 1) / G), low = n + (uint32_t)(r0 / G);  // what the last and the first token see
  const uint32_t window = c.window > 0 ? (uint32_t)c.window : 0xffffffffu;
  // the first position that any row sees (a length behind the table's end: every row sees its own position, which has no page, and is NaN, whatever
  // there is before)
  const uint32_t begin = (long long)n >= (long long)c.wide * c.page ? low : low >= window ? low + 1u - window : 0u;
  // tiles begin at multiples of 16, so that one of a page of a multiple of 16 lies within it; what a tile has before `begin` is not read
  const uint32_t first = begin / TILE_16 * TILE_16;
  const uint32_t tiles = idle ? 0u : (last - first) / TILE_16 + 1u, per = (tiles + parts - 1) / parts;
  const uint32_t t0 = part * per;
  const int mine = (int)min(tiles > t0 ? tiles - t0 : 0u, per) - warp;  // this warp takes t0 + warp, t0 + warp + W, ..
  const int steps = mine > 0 ? (mine + W - 1) / W : 0;
  const bool even = c.page % TILE_16 == 0;
  const int* pages = c.pages + (long long)b * c.wide;

  uint32_t pos = first + (t0 + warp) * TILE_16;  // of the tile that is fetched
  // The page of a tile's positions, a lane a position, is asked for a tile ahead: it is there when the tile's keys are to be fetched.
  int ahead = -1;
  uint32_t ahead_off = 0;
  auto lookup = [&](uint32_t from) {
    const uint32_t p = from + (lane & 15), slot = p / (uint32_t)c.page;
    ahead_off = p - slot * (uint32_t)c.page;
    ahead = p <= last && slot < (uint32_t)c.wide ? pages[slot] : -1;
  };
  // where the tile is: one base for all of it, or each position's own (held by the lane of that number; 0: seen by no row, 1: in the pool, 2: of the call)
  bool whole = false;
  long long base = 0, at = 0;
  int kind = 0;
  uint32_t missing = 0;  // positions without a page, a bit each
  auto locate = [&]() {
    const bool valid = (unsigned)ahead < (unsigned)c.n_pages;
    const uint32_t p = pos + (lane & 15);
    at = valid ? (long long)ahead * c.pool_p + (long long)ahead_off * c.pool_t + hkv * c.pool_h : 0;
    kind = p > last || p < begin ? 0 : !valid ? -1 : p >= n ? 2 : 1;
    missing = 0;
    whole = even && __all_sync(0xffffffffu, kind == 1);
    if (whole) {
      base = __shfl_sync(0xffffffffu, at, 0);
      return;
    }
    missing = __ballot_sync(0xffffffffu, kind == -1) & 0xffffu;
    // a token is added by the block that has its first row: that row sees it, whatever the window
    if (__any_sync(0xffffffffu, kind == 2)) {
      for (int i = 0; i < TILE_16; ++i) {
        const long long a = __shfl_sync(0xffffffffu, at, i), token = (long long)pos + i - n, own_row = token * G;
        if (__shfl_sync(0xffffffffu, kind, i) == 2 && own_row >= r0 && own_row < r0 + nr) {
          const T *ks = new_k + b * c.k.b + token * c.k.t + hkv * c.k.h, *vs = new_v + b * c.v.b + token * c.v.t + hkv * c.v.h;
          for (int d = lane * 8; d < c.D; d += 256) {
            *reinterpret_cast<uint4*>(pool_k + a + d) = *reinterpret_cast<const uint4*>(ks + d);
            *reinterpret_cast<uint4*>(pool_v + a + d) = *reinterpret_cast<const uint4*>(vs + d);
          }
        }
      }
    }
  };
  const T* const zeros = reinterpret_cast<const T*>(zero_row);
  auto row_of = [&](const T* pool, const T* fresh, const Strides& s, int i) -> const T* {
    const long long a = __shfl_sync(0xffffffffu, at, i);
    const int kd = __shfl_sync(0xffffffffu, kind, i);
    return kd == 1 ? pool + a : kd == 2 ? fresh + b * s.b + ((long long)pos + i - n) * s.t + hkv * s.h : zeros;
  };
  uint4 kr[2][CH], vr[4][VH];
  const T *const pool_kl = pool_k + g * c.pool_t + t4 * 8, *const pool_vl = pool_v + 2 * t4 * c.pool_t + g * 8;  // this lane's place in a whole tile
  auto load_k = [&]() {
    if (FULL && whole) {
      const T *p = pool_kl + base, *p8 = p + 8 * c.pool_t;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        kr[0][i] = load_once(p + 32 * i);
        kr[1][i] = load_once(p8 + 32 * i);
      }
      return;
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const T* p = whole ? pool_k + base + (g + 8 * u) * c.pool_t : row_of(pool_k, new_k, c.k, g + 8 * u);
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int d = (t4 + 4 * i) * 8;
        kr[u][i] = load_once(FULL || d < c.D ? p + d : zeros);
      }
    }
  };
  auto load_v = [&]() {
    if (FULL && whole) {
      const T *p = pool_vl + base, *p8 = p + 8 * c.pool_t;
#pragma unroll
      for (int i = 0; i < VH; ++i) {
        vr[0][i] = load_once(p + 64 * i);
        vr[1][i] = load_once(p + c.pool_t + 64 * i);
        vr[2][i] = load_once(p8 + 64 * i);
        vr[3][i] = load_once(p8 + c.pool_t + 64 * i);
      }
      return;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int row = 2 * t4 + (u & 1) + (u >> 1) * 8;
      const T* p = whole ? pool_v + base + row * c.pool_t : row_of(pool_v, new_v, c.v, row);
#pragma unroll
      for (int i = 0; i < VH; ++i) {
        const int d = (g + 8 * i) * 8;
        vr[u][i] = load_once(FULL || d < c.D ? p + d : zeros);
      }
    }
  };
  if (steps > 0) {
    lookup(pos);
    locate();
    load_k();
    load_v();
    lookup(pos + W * TILE_16);
  }

  // the queries' rows g (and 8 further), read in the same chunks as the keys
  uint32_t qb[NT][CH][4];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int r = g + 8 * j, t = (r0 + r) / G, h = hkv * G + (r0 + r) % G;
    const uint16_t* from = reinterpret_cast<const uint16_t*>(q + b * c.q.b + t * c.q.t + h * c.q.h);
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = (t4 + 4 * i) * 8 + 2 * e;
        qb[j][i][e] = r < nr && d < c.D ? (uint32_t)from[d] | (uint32_t)from[d + 1] << 16 : 0u;
      }
  }
  const bool cap = c.cap > 0.f, slopes = c.slopes != nullptr;
  const float post = (cap ? c.cap : c.scale) * LOG2E, pre = cap ? c.scale / c.cap : 1.f;
  // rows 2t and 2t + 1 of each eight
  float slope[NT][2], m[NT][2], l[NT][2], o[NT][MT][4];
  uint32_t sees[NT][2];  // last position; rows that are none see as the first one, and are not stored
#pragma unroll
  for (int j = 0; j < NT; ++j) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int r = 8 * j + 2 * t4 + u;
      sees[j][u] = n + (uint32_t)((r0 + (r < nr ? r : 0)) / G);
      slope[j][u] = slopes && r < nr ? c.slopes[hkv * G + (r0 + r) % G] * LOG2E : 0.f;
      m[j][u] = -INFINITY;
      l[j][u] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[j][i][e] = 0.f;
  }

  for (int step = 0; step < steps; ++step) {
    const uint32_t p0 = pos, gone = missing;
    float s[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[j][e] = 0.f;
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        mma<T>(s[j], kr[0][i].x, kr[1][i].x, kr[0][i].y, kr[1][i].y, qb[j][i][0], qb[j][i][1]);
        mma<T>(s[j], kr[0][i].z, kr[1][i].z, kr[0][i].w, kr[1][i].w, qb[j][i][2], qb[j][i][3]);
      }
    // the values of this tile are on their way or there: its keys' registers take the next one's
    const bool more = step + 1 < steps;
    if (more) {
      pos += W * TILE_16;
      locate();
      load_k();
      lookup(pos + W * TILE_16);
    }
    const bool masked = p0 + TILE_16 - 1 > low || last - p0 >= window || gone != 0;  // some row does not see some position
    uint32_t pb[NT][2];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      if (cap) capped4(s[j], pre, post);
      else {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[j][e] *= post;
      }
      if (slopes) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[j][e] = fmaf(-slope[j][e & 1], (float)(int)(sees[j][e & 1] - (p0 + g + 8 * (e >> 1))), s[j][e]);
      }
      if (masked) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = g + 8 * (e >> 1);
          const uint32_t p = p0 + i, to = sees[j][e & 1];
          if (gone >> i & 1u) s[j][e] = NAN;
          if (p > to || to - p >= window) s[j][e] = -INFINITY;
        }
      }
      float top[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        top[u] = fmaxf(s[j][u], s[j][2 + u]);
        if (s[j][u] != s[j][u] || s[j][2 + u] != s[j][2 + u]) l[j][u] = NAN;  // the maximum alone would pass over it
      }
#pragma unroll
      for (int w = 4; w < 32; w <<= 1)
#pragma unroll
        for (int u = 0; u < 2; ++u) top[u] = fmaxf(top[u], __shfl_xor_sync(0xffffffffu, top[u], w));
      // O is rescaled only when a maximum has grown by more than 2^8: until then P fits its type as it is
      if (__any_sync(0xffffffffu, top[0] > m[j][0] + 8.f || top[1] > m[j][1] + 8.f)) {
        float alpha[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float to = fmaxf(m[j][u], top[u]);
          alpha[u] = to == -INFINITY ? 1.f : ex2(m[j][u] - to);
          m[j][u] = to;
          l[j][u] *= alpha[u];
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[j][i][e] *= alpha[e & 1];
      }
      const float base0 = m[j][0] == -INFINITY ? 0.f : m[j][0], base1 = m[j][1] == -INFINITY ? 0.f : m[j][1];
#pragma unroll
      for (int k = 0; k < 2; ++k) {  // positions g and g + 8
        const float x = ex2(s[j][2 * k] - base0), y = ex2(s[j][2 * k + 1] - base1);
        l[j][0] += x;
        l[j][1] += y;
        pb[j][k] = transpose8(pair16(x, y, T()));
      }
    }
    // columns of a product's 16 rows: (DP = 128) 8 g + i and 64 further, (DP = 64) 8 g + 2 i and the next
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      uint32_t a[4];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int col = VH == 2 ? i : 2 * i + half, chunk = VH == 2 ? half : 0;
        const uint32_t sel = col & 1 ? 0x7632u : 0x5410u;
        const uint32_t w[4] = {(&vr[0][chunk].x)[col >> 1], (&vr[1][chunk].x)[col >> 1], (&vr[2][chunk].x)[col >> 1], (&vr[3][chunk].x)[col >> 1]};
        a[half] = __byte_perm(w[0], w[1], sel);
        a[2 + half] = __byte_perm(w[2], w[3], sel);
      }
#pragma unroll
      for (int j = 0; j < NT; ++j) mma<T>(o[j][i], a[0], a[1], a[2], a[3], pb[j][0], pb[j][1]);
    }
    if (more) load_v();
  }

  // the warps join: each leaves its part, the block adds them up relative to the largest maximum
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int w = 4; w < 32; w <<= 1) l[j][u] += __shfl_xor_sync(0xffffffffu, l[j][u], w);
      const int r = 8 * j + 2 * t4 + u;
      if (g == 0) {
        s_m[warp * ROWS_ + r] = m[j][u];
        s_l[warp * ROWS_ + r] = l[j][u];
      }
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int half = 0; half < 2; ++half) s_own[(warp * ROWS_ + r) * PITCH + (VH == 2 ? 8 * g + i + 64 * half : 8 * g + 2 * i + half)] = o[j][i][2 * half + u];
    }
  __syncthreads();
  if (tid < ROWS_) {
    float top = -INFINITY, sum = 0.f;
    for (int w = 0; w < W; ++w) top = fmaxf(top, s_m[w * ROWS_ + tid]);
    const float base_m = top == -INFINITY ? 0.f : top;
    for (int w = 0; w < W; ++w) {
      const float f = ex2(s_m[w * ROWS_ + tid] - base_m);
      s_f[w * ROWS_ + tid] = f;
      sum = fmaf(s_l[w * ROWS_ + tid], f, sum);
    }
    s_m[tid] = top;  // the block's own, over those of its first warp
    s_l[tid] = sum;
    if (!joined) ws.sums[((long long)unit * parts + part) * ROWS_ + tid] = make_float2(top, sum);
  }
  __syncthreads();
  for (int e = tid; e < nr * DP; e += W * 32) {
    const int r = e / DP, d = e % DP;
    float x = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) x = fmaf(s_own[(w * ROWS_ + r) * PITCH + d], s_f[w * ROWS_ + r], x);
    if (joined) s_part[r * PITCH + d] = x;
    else ws.rows[(((long long)unit * parts + part) * ROWS_ + r) * DP + d] = x;
  }
  if (!joined) return;
  cluster.sync();
  // and the blocks of the cluster: each makes its share of the result from everybody's parts
  for (int e = part * W * 32 + tid; e < nr * DP; e += parts * W * 32) {
    const int r = e / DP, d = e % DP;
    float top = -INFINITY, sum = 0.f, x = 0.f;
    for (int i = 0; i < parts; ++i) top = fmaxf(top, cluster.map_shared_rank(s_m, i)[r]);
    const float base_m = top == -INFINITY ? 0.f : top;
    for (int i = 0; i < parts; ++i) {
      const float f = ex2(cluster.map_shared_rank(s_m, i)[r] - base_m);
      sum = fmaf(cluster.map_shared_rank(s_l, i)[r], f, sum);
      x = fmaf(cluster.map_shared_rank(s_part, i)[r * PITCH + d], f, x);
    }
    const int t = (r0 + r) / G, h = hkv * G + (r0 + r) % G;
    if (d < c.D) out[(((long long)b * c.T + t) * c.H + h) * c.D + d] = from_f32<T>(sum == 0.f ? 0.f : x / sum);
  }
  cluster.sync();  // nobody leaves while its part is read
}

// A block a row of a unit: the parts' sums and rows, in order.
template <typename T, int DP, int NT>
__global__ void __launch_bounds__(DP) join_kernel(const Cache c, const Parts ws, T* out) {
  constexpr int ROWS_ = 8 * NT;
  const int G = c.H / c.Hkv, rows = c.T * G, row_tiles = (rows + ROWS_ - 1) / ROWS_;
  const int unit = blockIdx.x / ROWS_, r = blockIdx.x % ROWS_, rt = unit % row_tiles, hkv = unit / row_tiles % c.Hkv, b = unit / row_tiles / c.Hkv, d = threadIdx.x;
  const int row = rt * ROWS_ + r;
  if (row >= rows || d >= c.D) return;
  const float2* sums = ws.sums + (long long)unit * ws.count * ROWS_ + r;
  const float* from = ws.rows + ((long long)unit * ws.count * ROWS_ + r) * DP + d;
  float top = -INFINITY, sum = 0.f, x = 0.f;
  for (int i = 0; i < ws.count; ++i) top = fmaxf(top, sums[i * ROWS_].x);
  const float base = top == -INFINITY ? 0.f : top;
  for (int i = 0; i < ws.count; ++i) {
    const float2 v = sums[i * ROWS_];
    const float f = ex2(v.x - base);
    sum = fmaf(v.y, f, sum);
    x = fmaf(from[(long long)i * ROWS_ * DP], f, x);
  }
  const int t = row / G, h = hkv * G + row % G;
  out[(((long long)b * c.T + t) * c.H + h) * c.D + d] = from_f32<T>(sum == 0.f ? 0.f : x / sum);
}

template <typename T>
bool vectors(const void* p, long long a, long long b, long long c, int D) {
  constexpr int V = 16 / sizeof(T);
  return D % V == 0 && a % V == 0 && b % V == 0 && c % V == 0 && ((uintptr_t)p & 15) == 0;
}

template <typename... A>
void launch_parts(void (*kernel)(A...), long long blocks, int cluster, int threads, int smem, cudaStream_t stream, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)cluster;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Parts that a unit (a sequence, a key head, a tile of rows) is split into.
struct Split {
  long long units;
  int cluster;  // parts that join in a cluster
  int spread;   // more parts than a cluster has, which join through memory; 0: none
};
Split split_of(const Cache& c, bool tensor) {
  const long long rows = (long long)c.T * (c.H / c.Hkv), pairs = (long long)c.B * c.Hkv;
  Split s{pairs * (tensor && rows <= 8 ? 1 : (rows + 15) / 16), 1, 0};
  // positions that a row may see, where the table is full
  const long long full = (long long)c.wide * c.page, seen = c.window > 0 && c.window + (long long)c.T < full ? c.window + (long long)c.T : full;
  const long long most = (seen + 127) / 128;  // at least 128 positions a part
  const int sms = kb_sm_count();
  // clusters: as many parts as give every SM about four blocks, which evens out sequences of different lengths (64 sequences of 200 to 4000: 122 us,
  // whole 135 us).  Once there is a block for every SM a further part has to be worth its start: 1024 positions (16 sequences within a window of 1024: 40 us
  // in one part, 49 us in two).
  while (s.cluster < 8 && s.cluster * 2 <= most && s.units * s.cluster < 4ll * sms && (s.units * s.cluster < sms || s.cluster * 2048ll <= seen)) s.cluster *= 2;
  const int fit = tensor ? 3 : 2;  // blocks an SM
  if (s.cluster == 8 && s.units * 8 < (long long)fit * sms && most > 8) {
    // Few long sequences: one wave of three blocks an SM (two of the plain kernel's).  (Clusters of eight large blocks, of which the chip holds no more than about half as
    // many as its SMs would allow, took twice the time.)
    const long long want = (long long)fit * sms / s.units;
    s.spread = (int)(want < most ? want : most);
    if (s.spread > 8) s.cluster = 1;
    else s.spread = 0;
  }
  return s;
}

// Rows that a unit's parts leave, and floats of the workspace of parts that join through memory.
int rows_of(const Cache& c, bool tensor) { return tensor && (long long)c.T * (c.H / c.Hkv) <= 8 ? 8 : 16; }
long long work_of(const Cache& c, const Split& s, bool tensor) { return s.units * s.spread * rows_of(c, tensor) * ((c.D <= 64 ? 64 : c.D <= 128 ? 128 : 256) + 2); }

template <typename T, int DP>
int launch_cache(const Cache& c, const void* q, const void* k, const void* v, void* pk, void* pv, void* out, float* work, long long floats, bool tensor, cudaStream_t stream) {
  Split s = split_of(c, tensor);
  if (s.spread > 0 && work_of(c, s, tensor) > floats) {  // asked for on another kind of device
    s.spread = 0;
    s.cluster = 8;
  }
  Parts ws{nullptr, nullptr, s.spread};
  if (s.spread > 0) {
    ws.sums = reinterpret_cast<float2*>(work);
    ws.rows = work + 2 * s.units * s.spread * rows_of(c, tensor);
  }
  if constexpr (sizeof(T) == 2 && DP <= 128) {
    if (tensor) {
      const bool one = (long long)c.T * (c.H / c.Hkv) <= 8;
      const long long blocks = s.units * (s.spread > 0 ? s.spread : s.cluster);
#define KB_LAUNCH(NT, FULL) \
  launch_parts(cache_kernel_16<T, DP, NT, FULL>, blocks, s.cluster, 128, 0, stream, c, (const T*)q, (const T*)k, (const T*)v, (T*)pk, (T*)pv, (T*)out, (const Parts)ws)
      if (c.D == DP) {
        if (one) KB_LAUNCH(1, true);
        else KB_LAUNCH(2, true);
      } else {
        if (one) KB_LAUNCH(1, false);
        else KB_LAUNCH(2, false);
      }
#undef KB_LAUNCH
      if (s.spread > 0) {
        if (one) join_kernel<T, DP, 1><<<(unsigned)(s.units * 8), DP, 0, stream>>>(c, ws, (T*)out);
        else join_kernel<T, DP, 2><<<(unsigned)(s.units * 16), DP, 0, stream>>>(c, ws, (T*)out);
      }
      return 0;
    }
  }
  constexpr int SMEM = CacheTile<DP>::FLOATS * 4;
  static bool attr[KB_MAX_DEVICES] = {false};
  if (!kb_allow_smem(cache_kernel<T, DP>, SMEM, attr)) {
    kb200_set_error("attention_cache: shared-memory limit");
    return -3;
  }
  const int vec = vectors<T>(k, c.k.t, c.k.h, c.k.b, c.D) && vectors<T>(v, c.v.t, c.v.h, c.v.b, c.D) && vectors<T>(pk, c.pool_p, c.pool_t, c.pool_h, c.D) &&
                  vectors<T>(pv, c.pool_p, c.pool_t, c.pool_h, c.D);
  launch_parts(cache_kernel<T, DP>, s.units * (s.spread > 0 ? s.spread : s.cluster), s.cluster, THREADS, SMEM, stream, c, (const T*)q, (const T*)k, (const T*)v, (T*)pk, (T*)pv, (T*)out,
               (const Parts)ws, vec);
  if (s.spread > 0) join_kernel<T, DP, 2><<<(unsigned)(s.units * 16), DP, 0, stream>>>(c, ws, (T*)out);
  return 0;
}

// Whether the tensor-core kernel takes the call.
bool tensor_cores(const Cache& c, int dtype, const void* k, const void* v, const void* pk, const void* pv) {
  return dtype != 0 && c.D <= 128 && vectors<__half>(k, c.k.t, c.k.h, c.k.b, c.D) && vectors<__half>(v, c.v.t, c.v.h, c.v.b, c.D) &&
         vectors<__half>(pk, c.pool_p, c.pool_t, c.pool_h, c.D) && vectors<__half>(pv, c.pool_p, c.pool_t, c.pool_h, c.D);
}

}  // namespace

// Floats of workspace that kb200_attention_cache may use at these sizes.
KB_API long long kb200_attention_cache_work(int B, int H, int Hkv, int T, int D, int page, int wide, int window) {
  Cache c{};
  c.B = B;
  c.H = H;
  c.Hkv = Hkv;
  c.T = T;
  c.D = D;
  c.page = page;
  c.wide = wide;
  c.window = window;
  if (B <= 0 || T <= 0 || Hkv <= 0 || H < Hkv || D <= 0 || D > 256) return 0;
  const long long plain = work_of(c, split_of(c, false), false), tensor = D <= 128 ? work_of(c, split_of(c, true), true) : 0;
  return plain > tensor ? plain : tensor;
}

// q [B, T, H, D], new_k and new_v [B, T, Hkv, D], pools [n_pages, page, Hkv, D] of common strides, unit stride on D; out [B, T, H, D] contiguous;
// pages [B, wide] and lengths [B] contiguous.  strides: q, k, v as (token, head, sequence), then the pools' (page, position, head).  work: `floats` of them, as
// many as kb200_attention_cache_work says.  dtype 0 float32, 1 bfloat16, 2 float16.
KB_API int kb200_attention_cache(const void* q, const void* new_k, const void* new_v, void* pool_k, void* pool_v, void* out, const int* pages, const int* lengths,
                                 const long long* strides, float* work, long long floats, int dtype, int B, int H, int Hkv, int T, int D, int n_pages, int page, int wide, float scale, float cap,
                                 const float* slopes, int window, cudaStream_t stream) {
  if (B <= 0 || T <= 0 || H <= 0 || Hkv <= 0 || H % Hkv || D <= 0 || D > 256 || n_pages <= 0 || page <= 0 || wide <= 0 || dtype < 0 || dtype > 2) {
    kb200_set_error("attention_cache: sizes out of range (heads of up to 256, query heads a multiple of key heads)");
    return -2;
  }
  const long long units = (long long)B * Hkv * (((long long)T * (H / Hkv) + 15) / 16);
  if ((long long)T * (H / Hkv) > (1 << 30) || units > 0x7ffffffll) {
    kb200_set_error("attention_cache: too many rows");
    return -2;
  }
  const Cache c{B, H, Hkv, T, D, n_pages, page, wide, strides[9], strides[10], strides[11], {strides[0], strides[1], strides[2]}, {strides[3], strides[4], strides[5]},
                {strides[6], strides[7], strides[8]}, pages, lengths, scale, cap, slopes, window};
  const bool tensor = tensor_cores(c, dtype, new_k, new_v, pool_k, pool_v);
  int rc;
#define KB_CACHE(TT)                                                                                     \
  (D <= 64    ? launch_cache<TT, 64>(c, q, new_k, new_v, pool_k, pool_v, out, work, floats, tensor, stream)      \
   : D <= 128 ? launch_cache<TT, 128>(c, q, new_k, new_v, pool_k, pool_v, out, work, floats, tensor, stream)     \
              : launch_cache<TT, 256>(c, q, new_k, new_v, pool_k, pool_v, out, work, floats, tensor, stream))
  rc = dtype == 0 ? KB_CACHE(float) : dtype == 1 ? KB_CACHE(__nv_bfloat16) : KB_CACHE(__half);
#undef KB_CACHE
  if (rc != 0) return rc;
  KB_CHECK_LAUNCH("attention_cache");
  return 0;
}
