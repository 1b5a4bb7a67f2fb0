// Attention of new tokens over a paged key/value cache, with their keys and values added to it in the same launch.
//
// The cache is two pools of pages, [P, page, Hkv, D] each; pages[b, n] names the pool's page that holds positions n * page .. of sequence b.
// A call brings T new tokens a sequence.  Their keys and values go to positions n .. n + T - 1 (n = lengths[b]), and the query of token t
// sees the positions up to n + t, within the window if there is one.  Scores are those of attention_rules.cuh: cap and slopes.
//
// A decoder's step reads each key and value once and does little else, so the cache's bytes bound it.  One sequence and key head is the
// work of a thread-block cluster: its CTAs take equal parts of the visible positions, each with a running maximum and sum, and join
// their parts through distributed shared memory: one launch, no workspace, and the same order of sums every time.  The T * H / Hkv rows
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
constexpr int ROWS = 16;   // rows of a CTA at most
constexpr int THREADS = 128;

template <int DP>
struct CacheTile {
  static constexpr int PITCH = DP + 4;
  static constexpr int FLOATS = ROWS * PITCH + KEYS * PITCH * 2 + ROWS * (KEYS + 1) + 3 * ROWS;
};

template <typename T, int DP>
__global__ void __launch_bounds__(THREADS) cache_kernel(const Cache c, const T* q, const T* new_k, const T* new_v, T* pool_k, T* pool_v, T* out, int vec) {
  constexpr int PITCH = CacheTile<DP>::PITCH, COLS = DP / THREADS > 0 ? DP / THREADS : 1;
  extern __shared__ __align__(16) float sm[];
  float *sQ = sm, *sK = sQ + ROWS * PITCH, *sV = sK + KEYS * PITCH, *sP = sV + KEYS * PITCH, *sM = sP + ROWS * (KEYS + 1), *sL = sM + ROWS, *sA = sL + ROWS;
  __shared__ int s_bad[KEYS];
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
  const int G = c.H / c.Hkv, rows = c.T * G, row_tiles = (rows + ROWS - 1) / ROWS;
  const int unit = (int)(blockIdx.x / parts), rt = unit % row_tiles, hkv = unit / row_tiles % c.Hkv, b = unit / row_tiles / c.Hkv;
  const int r0 = rt * ROWS, nr = min(ROWS, rows - r0);  // row r: token r / G, query head hkv * G + r % G
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const long long n = c.lengths[b];
  const long long last = n < 0 ? -1 : n + (r0 + nr - 1) / G;  // of the positions that any row sees
  const long long first = n < 0 ? 0 : c.window > 0 ? max(0ll, n + r0 / G - c.window + 1) : 0;
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

template <typename T>
bool vectors(const void* p, long long a, long long b, long long c, int D) {
  constexpr int V = 16 / sizeof(T);
  return D % V == 0 && a % V == 0 && b % V == 0 && c % V == 0 && ((uintptr_t)p & 15) == 0;
}

template <typename T, int DP>
int launch_cache(const Cache& c, const void* q, const void* k, const void* v, void* pk, void* pv, void* out, int parts, cudaStream_t stream) {
  constexpr int SMEM = CacheTile<DP>::FLOATS * 4;
  static bool attr[KB_MAX_DEVICES] = {false};
  if (!kb_allow_smem(cache_kernel<T, DP>, SMEM, attr)) {
    kb200_set_error("attention_cache: shared-memory limit");
    return -3;
  }
  const int vec = vectors<T>(k, c.k.t, c.k.h, c.k.b, c.D) && vectors<T>(v, c.v.t, c.v.h, c.v.b, c.D) && vectors<T>(pk, c.pool_p, c.pool_t, c.pool_h, c.D) &&
                  vectors<T>(pv, c.pool_p, c.pool_t, c.pool_h, c.D);
  const int row_tiles = (c.T * (c.H / c.Hkv) + ROWS - 1) / ROWS;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((long long)c.B * c.Hkv * row_tiles * parts));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)parts;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, cache_kernel<T, DP>, c, (const T*)q, (const T*)k, (const T*)v, (T*)pk, (T*)pv, (T*)out, vec);
  return 0;
}

}  // namespace

// q [B, T, H, D], new_k and new_v [B, T, Hkv, D], pools [n_pages, page, Hkv, D] of common strides, unit stride on D; out [B, T, H, D] contiguous;
// pages [B, wide] and lengths [B] contiguous.  strides: q, k, v as (token, head, sequence), then the pools' (page, position, head).  dtype 0 float32,
// 1 bfloat16, 2 float16.
KB_API int kb200_attention_cache(const void* q, const void* new_k, const void* new_v, void* pool_k, void* pool_v, void* out, const int* pages, const int* lengths,
                                 const long long* strides, int dtype, int B, int H, int Hkv, int T, int D, int n_pages, int page, int wide, float scale, float cap,
                                 const float* slopes, int window, cudaStream_t stream) {
  if (B <= 0 || T <= 0 || H <= 0 || Hkv <= 0 || H % Hkv || D <= 0 || D > 256 || n_pages <= 0 || page <= 0 || wide <= 0 || dtype < 0 || dtype > 2) {
    kb200_set_error("attention_cache: sizes out of range (heads of up to 256, query heads a multiple of key heads)");
    return -2;
  }
  const long long units = (long long)B * Hkv * (((long long)T * (H / Hkv) + ROWS - 1) / ROWS);
  if ((long long)T * (H / Hkv) > (1 << 30) || units > 0x7ffffffll) {
    kb200_set_error("attention_cache: too many rows");
    return -2;
  }
  const Cache c{B, H, Hkv, T, D, n_pages, page, wide, strides[9], strides[10], strides[11], {strides[0], strides[1], strides[2]}, {strides[3], strides[4], strides[5]},
                {strides[6], strides[7], strides[8]}, pages, lengths, scale, cap, slopes, window};
  // as many parts as fill the chip about twice, each of at least four tiles where the table is full
  const long long most = ((long long)wide * page + 4 * KEYS - 1) / (4 * KEYS);
  int parts = 1;
  while (parts < 8 && parts * 2 <= most && units * parts < 2ll * kb_sm_count()) parts *= 2;
  int rc;
#define KB_CACHE(TT) (D <= 64 ? launch_cache<TT, 64>(c, q, new_k, new_v, pool_k, pool_v, out, parts, stream) : D <= 128 ? launch_cache<TT, 128>(c, q, new_k, new_v, pool_k, pool_v, out, parts, stream) : launch_cache<TT, 256>(c, q, new_k, new_v, pool_k, pool_v, out, parts, stream))
  rc = dtype == 0 ? KB_CACHE(float) : dtype == 1 ? KB_CACHE(__nv_bfloat16) : KB_CACHE(__half);
#undef KB_CACHE
  if (rc != 0) return rc;
  KB_CHECK_LAUNCH("attention_cache");
  return 0;
}
