// Group normalisation of [N, C] rows per scene, with the activation behind it:
//     mean, var of (rows of the scene) x (channels of the group);  xhat = (x - mean) / sqrt(var + eps)
//     y = act(gamma xhat + beta)                                   act: none, ReLU, SiLU, GELU
// and its gradients, with dz = dy act'(gamma xhat + beta) and M values in a (scene, group):
//     dbeta = sum dz,  dgamma = sum dz xhat,  dx = (gamma dz - sum(gamma dz) / M - xhat sum(gamma dz xhat) / M) / std.
//
// Bound by HBM where the rows are larger than L2, by L2 and latency below.  Each direction looks at the rows twice, first for
// sums, then to write the result, in ONE launch: tiles of both looks are items that blocks claim in order, a scene's second look
// following its first one at a distance of `lag` tiles, so that it finds the rows in L2 while other blocks are at the next
// scene's first look: HBM sees the rows once (those of scenes that do not fit L2 twice) and no multiprocessor waits between
// looks.  (A launch a look and group of scenes of 48 MB took 529 us instead of the 869 of many short tiles for 8 x 150 000 rows
// of 96 channels fp16, forward and backward, of which the launches' starts and ends were half.)  This one takes 163 + 256 us there,
// 2.8 and 2.7 TB/s of what has to move: neither HBM (30 to 43 %) nor the issue slots (31 to 40 %) are full, the 16 warps that 128
// registers leave a multiprocessor wait for an item's loads and its turn.  More warps of fewer registers, other distances between
// the looks and other tile sizes took as long or longer.  4 x 60 000 rows x 64 channels bf16 with ReLU: 31 + 46 us.
// A thread owns 16 bytes of channels and walks the rows of a tile of its scene; a tile leaves one mean and one sum of squared
// distances from it per group (backward: two sums, and two per channel); the block that leaves a scene's last tile puts the
// tiles together, in their order and in double, and raises the scene's flag: the same bits on every run.
// What an item waits for has been claimed before it, by blocks that are running: there is always one that can go on.  Waits are
// bounded all the same; one that runs out sets the status word, and what could not be computed is filled with NaN: all of the
// results of a launch that finds the word set by an earlier one.
// Variances are never differences of large numbers: a thread's few rows of a tile have a mean of their own, about the first of
// them, and means are put together by their differences: neither a row far from all others nor a mean that is large against the
// spread costs them precision.  Of a large mean its own rounding to fp32 is left in x - mean: up to 2^-24 |mean| / std in a
// result before gamma (nothing where the mean is a number of fp32, as in a constant group).
#include <string.h>

#include <type_traits>

#include "tcgen05_common.cuh"

namespace {

constexpr int THREADS = 256;
constexpr int BLOCKS_FORWARD = 2, BLOCKS_BACKWARD = 2;   // of a multiprocessor (128 registers a thread)
// Scenes of a launch, half of the 32 KB of parameters that one may have.  128, 320 and 1280 of them: 1 000 scenes of 60 rows x 64
// channels fp16 in 108, 77 and 51 us, 4 000 of 30 rows in 428, 254 and 187; one scene of 20 000 rows in 19.8 with each, of 2 000 in
// 15.5, 15.9 and 16.4 of a captured graph and in 26, 28 and 20 as calls.
constexpr int SCENES = 1280;
constexpr int MAX_C = 4096;

enum Act { NONE = 0, RELU = 1, SILU = 2, GELU = 3 };

struct Scenes {
  int count;               // with rows
  int scene[SCENES];       // its place among all of them
  int row0[SCENES + 1];    // first row, from the launch's first row on
  int tile0[SCENES + 1];   // first tile
};

// What the blocks of a launch share, all zero before and after it.
struct Sync {
  int ticket, done, scenes;      // items claimed, blocks that have ended, scenes whose sums are complete
  int tiles[SCENES], flag[SCENES];
};

struct Params {
  const void* x;
  const void* dy;
  void* out;              // y or dx
  const float* gamma;     // null: 1
  const float* beta;      // null: 0
  float* mean;            // [scenes][G]
  float* rstd;
  float2* part;           // [tiles][G]: (mean, sum of squared distances); backward: (sum gamma dz, sum gamma dz xhat)
  float2* whole;          // [scenes][G] of all tiles: (mean, 1 / std); backward: the two sums over M
  float* channels;        // [tiles][2][C] backward: sum dz, sum dz xhat (null: not wanted)
  float* sums;            // [2][C] of all tiles: added to from the second launch on
  int64_t x_ld, dy_ld;
  int C, G, per;          // per: channels of a group
  int rows, each;         // rows of a tile, and of each of its threads
  int tiles, lag, items;
  int add;                // `sums` has something already
  float eps;
  Sync* sync;
  int32_t* dev_status;
};

template <typename T, int V> struct alignas(V * sizeof(T)) Piece { T v[V]; };
template <typename T, int V> __device__ __forceinline__ Piece<T, V> load_piece(const T* p) {
  Piece<T, V> q;
  if constexpr (V * sizeof(T) == 16) *reinterpret_cast<uint4*>(q.v) = __ldg(reinterpret_cast<const uint4*>(p));
  else
    for (int i = 0; i < V; ++i) q.v[i] = p[i];
  return q;
}
// Rounded two at a time (a conversion of one number goes through the slow pipe of the special functions).
template <typename T, int V> __device__ __forceinline__ Piece<T, V> rounded(const float2 (&f)[(V + 1) / 2]) {
  Piece<T, V> q;
#pragma unroll
  for (int i = 0; i < (V + 1) / 2; ++i) {
    if constexpr (V == 1) q.v[0] = wcn_from_float<T>(f[i].x);
    else if constexpr (std::is_same<T, __half>::value) *reinterpret_cast<__half2*>(q.v + 2 * i) = __float22half2_rn(f[i]);
    else if constexpr (std::is_same<T, __nv_bfloat16>::value) *reinterpret_cast<__nv_bfloat162*>(q.v + 2 * i) = __float22bfloat162_rn(f[i]);
    else { q.v[2 * i] = f[i].x; q.v[2 * i + 1] = f[i].y; }
  }
  return q;
}

// The last look at a piece and what is written: not kept in L2 at the cost of rows that are to be looked at again.
template <typename T, int V> __device__ __forceinline__ Piece<T, V> load_last(const T* p) {
  Piece<T, V> q;
  if constexpr (V * sizeof(T) == 16) *reinterpret_cast<uint4*>(q.v) = __ldcs(reinterpret_cast<const uint4*>(p));
  else
    for (int i = 0; i < V; ++i) q.v[i] = p[i];
  return q;
}
template <typename T, int V> __device__ __forceinline__ void store_piece(T* p, const Piece<T, V>& q) {
  if constexpr (V * sizeof(T) == 16) __stcs(reinterpret_cast<uint4*>(p), *reinterpret_cast<const uint4*>(q.v));
  else
    for (int i = 0; i < V; ++i) p[i] = q.v[i];
}

// Pairs of numbers, one instruction each.
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
template <typename T, int V> __device__ __forceinline__ float2 pair_of(const Piece<T, V>& q, int i) {
  if constexpr (V == 1) return make_float2(wcn_to_float<T>(q.v[0]), 0.f);
  else if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(q.v + 2 * i));
  else if constexpr (std::is_same<T, __nv_bfloat16>::value) return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(q.v + 2 * i));
  else return make_float2(q.v[2 * i], q.v[2 * i + 1]);
}
// Per-channel values of a piece, from channel c on.
template <int V> __device__ __forceinline__ float2 pair_at(const float* p, int c, float none) {
  return p ? make_float2(__ldg(p + c), V == 1 ? none : __ldg(p + c + (V > 1))) : both(none);
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float reciprocal_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 1 / (1 + exp(-z))
__device__ __forceinline__ float2 logistic(float2 z) {
  const float2 e = __fmul2_rn(z, both(-1.4426950408889634f));
  const float2 d = __fadd2_rn(both(1.f), make_float2(exp2_fast(e.x), exp2_fast(e.y)));
  return make_float2(reciprocal_fast(d.x), reciprocal_fast(d.y));
}
// (1 + erf(z / sqrt(2))) / 2
__device__ __forceinline__ float2 normal(float2 z) {
  const float2 h = __fmul2_rn(z, both(0.70710678118654752f));
  return __ffma2_rn(make_float2(erff(h.x), erff(h.y)), both(0.5f), both(0.5f));
}

template <int ACT> __device__ __forceinline__ float2 activate(float2 z) {
  if (ACT == RELU) return make_float2(z.x > 0.f || z.x != z.x ? z.x : 0.f, z.y > 0.f || z.y != z.y ? z.y : 0.f);
  if (ACT == SILU) return __fmul2_rn(z, logistic(z));
  if (ACT == GELU) return __fmul2_rn(z, normal(z));
  return z;
}
// dy act'(z)
template <int ACT> __device__ __forceinline__ float2 through(float2 dy, float2 z) {
  if (ACT == RELU) return make_float2(z.x > 0.f || z.x != z.x ? dy.x : 0.f, z.y > 0.f || z.y != z.y ? dy.y : 0.f);
  if (ACT == SILU) {
    const float2 p = logistic(z), q = __ffma2_rn(p, both(-1.f), both(1.f));
    return __fmul2_rn(dy, __fmul2_rn(p, __ffma2_rn(z, q, both(1.f))));
  }
  if (ACT == GELU) {
    const float2 e = __fmul2_rn(__fmul2_rn(z, z), both(-0.72134752044448170f));
    const float2 density = make_float2(0.3989422804014327f * exp2_fast(e.x), 0.3989422804014327f * exp2_fast(e.y));
    return __fmul2_rn(dy, __ffma2_rn(z, density, normal(z)));
  }
  return dy;
}

// The scene and the rows of a tile.
struct Tile { int scene, place, lo, hi, first, last; };   // scene of the launch, its place among all; first, last: its tiles
__device__ __forceinline__ Tile find_tile(const Scenes& s, int tile, int rows) {
  int at = 0;
  for (int hi = s.count; hi - at > 1;) {
    const int mid = (at + hi) / 2;
    if (s.tile0[mid] <= tile) at = mid; else hi = mid;
  }
  Tile t{at, s.scene[at], 0, 0, s.tile0[at], s.tile0[at + 1]};
  t.lo = s.row0[at] + (tile - t.first) * rows;
  t.hi = min(t.lo + rows, s.row0[at + 1]);
  return t;
}

// Places of the threads: `txs` pieces of channels side by side, `tys` rows.
struct Place {
  int txs, tys, tx, ty, pieces;
  __device__ __forceinline__ Place(int C, int V) {
    pieces = C / V;
    txs = min(pieces, THREADS);
    tys = THREADS / txs;
    tx = threadIdx.x % txs;
    ty = threadIdx.x / txs;
  }
};

// Sums of a value over the rows' threads, for each of the W channels side by side: as many neighbouring threads a channel as there
// are, V values each.  f(channel, y0, step, sum) is called by all threads that share a channel (y0, y0 + step, .. are theirs;
// sum adds over them), last with the threads of channels beyond W.
template <typename F> __device__ __forceinline__ void per_channel(int W, F&& f) {
  int share = 1;
  while (share < 32 && share * 2 * W <= THREADS) share *= 2;
  for (int c0 = 0; c0 < W; c0 += THREADS / share) f(c0 + (int)threadIdx.x / share, (int)threadIdx.x % share, share);
}
__device__ __forceinline__ float sum_over(float v, int share) {
  for (int o = share >> 1; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}
__device__ __forceinline__ double sum_over(double v, int share) {
  for (int o = share >> 1; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}
// f(group, lane, lanes) by as many neighbouring threads a group as there are, at most a warp.
template <typename F> __device__ __forceinline__ void per_group(int G, F&& f) {
  int width = 32;
  while (width > 1 && width * G > THREADS) width >>= 1;
  for (int g0 = 0; g0 < G; g0 += THREADS / width) f(g0 + (int)threadIdx.x / width, (int)threadIdx.x % width, width);
}

// f(j, what load(j) gives) for a thread's rows, U of them loaded while the U before are worked on.
template <int U, typename L, typename F> __device__ __forceinline__ void walk(int rows, L&& load, F&& f) {
  decltype(load(0)) a[U], b[U];
  int j = 0;
  if (rows >= U) {
#pragma unroll
    for (int u = 0; u < U; ++u) a[u] = load(u);
    for (;;) {
      const bool more = j + 2 * U <= rows;
      if (more) {
#pragma unroll
        for (int u = 0; u < U; ++u) b[u] = load(j + U + u);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) f(j + u, a[u]);
      j += U;
      if (!more) break;
      const bool again = j + 2 * U <= rows;
      if (again) {
#pragma unroll
        for (int u = 0; u < U; ++u) a[u] = load(j + U + u);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) f(j + u, b[u]);
      j += U;
      if (!again) break;
    }
  }
  if (j == rows) return;
#pragma unroll
  for (int u = 0; u < U - 1; ++u)
    if (j + u < rows) a[u] = load(j + u);
#pragma unroll
  for (int u = 0; u < U - 1; ++u)
    if (j + u < rows) f(j + u, a[u]);
}
// Rows of a thread in a tile of n.
__device__ __forceinline__ int rows_of(const Params& p, const Place& at, int n) {
  return n == p.rows ? p.each : n / at.tys + (at.ty < n % at.tys);
}

__device__ __forceinline__ int load_acquire(const int* p) {
  int v;
  asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void store_release(int* p, int v) { asm volatile("st.release.gpu.global.s32 [%0], %1;" ::"l"(p), "r"(v) : "memory"); }

// Waits (one thread) until *p is `want`; false: the limit has passed, here or elsewhere.
__device__ __noinline__ bool wait_for(const int* p, int want, int32_t* dev_status) {
  const long long t0 = clock64();
  for (int i = 0;; ++i) {
    if (load_acquire(p) == want) return true;
    if ((i & 255) == 255) {
      if (*(volatile int32_t*)dev_status == (int)WCN_ERR_WAIT_EXPIRED) return false;
      if (clock64() - t0 > kWaitCycles) {
        atomicExch(dev_status, (int)WCN_ERR_WAIT_EXPIRED);
        return false;
      }
    }
  }
}

template <typename T, int V>
__device__ __forceinline__ void tile_stats(const Params& p, const Place& at, const Tile& t, int tile, float* smem) {
  const int W = at.txs * V;                       // channels side by side
  float* const s_mean = smem;                     // [tys][W]
  float* const s_m2 = smem + at.tys * W;          // [tys][W]
  float* const c_mean = s_m2 + at.tys * W;        // [C]
  float* const c_m2 = c_mean + p.C;               // [C]
  const int n_tile = t.hi - t.lo, n_each = n_tile == p.rows ? p.each : n_tile / at.tys, n_more = n_tile - n_each * at.tys;   // rows of a thread: one more for the first
  const T* const x = reinterpret_cast<const T*>(p.x);
  for (int pc = at.tx; pc - at.tx < at.pieces; pc += at.txs) {
    if (at.ty < at.tys && pc < at.pieces) {
      // About the thread's first row: at most 67 rows, of which a far first one spoils the others' distances by no more than
      // its own distance counts for.
      constexpr int P = (V + 1) / 2;
      float2 first[P], s1[P], s2[P];     // (its negative)
      const int rows = rows_of(p, at, n_tile);
      const int64_t step = (int64_t)at.tys * p.x_ld;
      const T* const from = x + (int64_t)(t.lo + at.ty) * p.x_ld + pc * V;
#pragma unroll
      for (int i = 0; i < P; ++i) first[i] = s1[i] = s2[i] = both(0.f);
      if (rows) {
        const Piece<T, V> q = load_piece<T, V>(from);
#pragma unroll
        for (int i = 0; i < P; ++i) first[i] = __fmul2_rn(pair_of<T, V>(q, i), both(-1.f));
      }
      walk<4>(rows, [&](int j) { return load_piece<T, V>(from + j * step); }, [&](int, const Piece<T, V>& q) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
          const float2 d = __fadd2_rn(pair_of<T, V>(q, i), first[i]);
          s1[i] = __fadd2_rn(s1[i], d);
          s2[i] = __ffma2_rn(d, d, s2[i]);
        }
      });
      const float inv = rows ? 1.f / (float)rows : 0.f;
      auto leave = [&](int c, float first, float s1, float s2) {
        const float d = s1 * inv;
        s_mean[at.ty * W + at.tx * V + c] = d - first;
        s_m2[at.ty * W + at.tx * V + c] = fmaxf(fmaf(-s1, d, s2), 0.f) + (s1 - s1);   // (NaN stays NaN)
      };
#pragma unroll
      for (int i = 0; i < P; ++i) {
        leave(2 * i, first[i].x, s1[i].x, s2[i].x);
        if (V > 1) leave(2 * i + 1, first[i].y, s1[i].y, s2[i].y);
      }
    }
    __syncthreads();
    const int c0 = (pc - at.tx) * V;
    per_channel(W, [&](int c, int y0, int share) {
      const bool live = c < W && c0 + c < p.C;
      float sum = 0.f, m2 = 0.f;
      if (live)
        for (int y = y0; y < at.tys; y += share) sum = fmaf(s_mean[y * W + c], (float)(n_each + (y < n_more)), sum);
      const float m = sum_over(sum, share) / (float)n_tile;
      if (live)
        for (int y = y0; y < at.tys; y += share) {
          const float d = s_mean[y * W + c] - m;
          m2 += fmaf(d * d, (float)(n_each + (y < n_more)), s_m2[y * W + c]);
        }
      m2 = sum_over(m2, share);
      if (live && y0 == 0) {
        c_mean[c0 + c] = m;
        c_m2[c0 + c] = m2;
      }
    });
    __syncthreads();
  }
  per_group(p.G, [&](int g, int lane, int width) {
    float sum = 0.f, m2 = 0.f;
    if (g < p.G)
      for (int c = lane; c < p.per; c += width) sum += c_mean[g * p.per + c];
    const float m = sum_over(sum, width) / (float)p.per;
    if (g < p.G)
      for (int c = lane; c < p.per; c += width) {
        const float d = c_mean[g * p.per + c] - m;
        m2 += fmaf(d * d, (float)n_tile, c_m2[g * p.per + c]);
      }
    m2 = sum_over(m2, width);
    if (g < p.G && lane == 0) p.part[(int64_t)tile * p.G + g] = make_float2(m, m2);
  });
}

// The tiles of a scene together: f(group, lane, lanes) leaves the group's values in `whole`.
template <typename T, int V>
__device__ __forceinline__ void join_stats(const Params& p, const Tile& t, int n_scene) {
  const int n_last = n_scene - (t.last - t.first - 1) * p.rows;
  per_group(p.G, [&](int g, int lane, int width) {
    // in one pass, about the first tile's mean: what the tiles' means differ by is no more than the spread
    double d1 = 0, d2 = 0;
    float about = 0.f;
    if (g < p.G) {
      about = __ldcg(&p.part[(int64_t)t.first * p.G + g]).x;
#pragma unroll 8
      for (int i = t.first + lane; i < t.last; i += width) {
        const float2 v = __ldcg(&p.part[(int64_t)i * p.G + g]);
        const double k = (double)(i == t.last - 1 ? n_last : p.rows), d = (double)v.x - (double)about;
        d1 += k * d;
        d2 += (double)v.y + k * d * d * p.per;
      }
    }
    const double n = (double)n_scene;
    d1 = sum_over(d1, width) / n;
    d2 = sum_over(d2, width);
    if (g < p.G && lane == 0) {
      const double var = d2 / (n * p.per) - d1 * d1;
      const float mean = (float)((double)about + d1), rstd = (float)(1.0 / sqrt((var < 0 ? 0 : var) + (double)p.eps));
      p.whole[(int64_t)t.scene * p.G + g] = make_float2(mean, rstd);
      if (p.mean) {
        p.mean[(int64_t)t.place * p.G + g] = mean;
        p.rstd[(int64_t)t.place * p.G + g] = rstd;
      }
    }
  });
}

__device__ __forceinline__ void join_grad_sums(const Params& p, const Tile& t, int n_scene) {
  per_group(p.G, [&](int g, int lane, int width) {
    double a = 0, b = 0;
    if (g < p.G)
#pragma unroll 8
      for (int i = t.first + lane; i < t.last; i += width) {
        const float2 v = __ldcg(&p.part[(int64_t)i * p.G + g]);
        a += (double)v.x;
        b += (double)v.y;
      }
    a = sum_over(a, width);
    b = sum_over(b, width);
    if (g < p.G && lane == 0) {
      const double inv = 1.0 / ((double)n_scene * p.per);
      p.whole[(int64_t)t.scene * p.G + g] = make_float2((float)(a * inv), (float)(b * inv));
    }
  });
}

// x - mean, before anything is scaled: x / std - mean / std would be a difference of numbers that are rounded at the size of
// mean / std (of a constant group of 1000 with eps 1e-5: 3e5, and results off by 0.016 where they are beta).
__device__ __forceinline__ float2 less(float2 x, float2 mean) { return __fadd2_rn(x, make_float2(-mean.x, -mean.y)); }
// A piece has SUB groups side by side (V / SUB channels of one group each; V: any).
// The values of a pair of channels, which may be of two of a piece's SUB groups.
template <int V, int SUB> __device__ __forceinline__ float2 of_pair(const float (&v)[SUB], int i) {
  return make_float2(v[2 * i * SUB / V], v[V == 1 ? 0 : (2 * i + 1) * SUB / V]);
}

// ready(): waits for the scene's sums (all threads); what does not depend on them is asked for before.
template <typename T, int V, int ACT, int SUB, typename R>
__device__ __forceinline__ void tile_apply(const Params& p, const Place& at, const Tile& t, R&& ready) {
  constexpr int P = (V + 1) / 2;
  bool ok = false, asked = false;
  const int rows = rows_of(p, at, t.hi - t.lo);
  const int64_t step = (int64_t)at.tys * p.x_ld, out_step = (int64_t)at.tys * p.C;
  for (int pc = at.tx; pc < at.pieces || !asked; pc += at.txs) {
    const int c0 = min(pc, at.pieces - 1) * V;
    const T* const from = reinterpret_cast<const T*>(p.x) + (int64_t)(t.lo + at.ty) * p.x_ld + pc * V;
    T* const to = reinterpret_cast<T*>(p.out) + (int64_t)(t.lo + at.ty) * p.C + pc * V;
    float mean[SUB], rstd[SUB];
    float2 scale[P], beta[P];
#pragma unroll
    for (int i = 0; i < P; ++i) {
      scale[i] = pair_at<V>(p.gamma, c0 + 2 * i, 1.f);
      beta[i] = pair_at<V>(p.beta, c0 + 2 * i, 0.f);
    }
    if (!asked) ok = ready();
    asked = true;
    if (at.ty >= at.tys || pc >= at.pieces) return;
#pragma unroll
    for (int k = 0; k < SUB; ++k) {
      const int g = (pc * V + k * (V / SUB)) / p.per;
      const float2 v = ok ? __ldcg(&p.whole[(int64_t)t.scene * p.G + g]) : make_float2(__int_as_float(0x7FC00000), 1.f);
      mean[k] = v.x;
      rstd[k] = v.y;
    }
#pragma unroll
    for (int i = 0; i < P; ++i) scale[i] = __fmul2_rn(of_pair<V, SUB>(rstd, i), scale[i]);
    walk<4>(rows, [&](int j) { return load_last<T, V>(from + j * step); }, [&](int j, const Piece<T, V>& q) {
      float2 o[P];
#pragma unroll
      for (int i = 0; i < P; ++i) o[i] = activate<ACT>(__ffma2_rn(less(pair_of<T, V>(q, i), of_pair<V, SUB>(mean, i)), scale[i], beta[i]));
      store_piece<T, V>(to + j * out_step, rounded<T, V>(o));
    });
  }
}

template <typename T, int V> struct Pair { Piece<T, V> x, dy; };

template <typename T, int V, int ACT, int SUB>
__device__ __forceinline__ void tile_grad_sums(const Params& p, const Place& at, const Tile& t, int tile, float* smem) {
  const int W = at.txs * V;
  float* const s_a = smem;                    // [tys][W]
  float* const s_b = smem + at.tys * W;       // [tys][W]
  float* const c_a = s_b + at.tys * W;        // [C] gamma dz
  float* const c_b = c_a + p.C;               // [C] gamma dz xhat
  for (int pc = at.tx; pc - at.tx < at.pieces; pc += at.txs) {
    if (at.ty < at.tys && pc < at.pieces) {
      const T* const x = reinterpret_cast<const T*>(p.x) + (int64_t)(t.lo + at.ty) * p.x_ld + pc * V;
      const T* const dy = reinterpret_cast<const T*>(p.dy) + (int64_t)(t.lo + at.ty) * p.dy_ld + pc * V;
      const int64_t step = (int64_t)at.tys * p.x_ld, dy_step = (int64_t)at.tys * p.dy_ld;
      constexpr int P = (V + 1) / 2;
      float2 a[P], b[P], scale[P], beta[P];   // (b: of x - mean, multiplied by 1 / std at the end)
      float mean[SUB], rstd[SUB];
#pragma unroll
      for (int k = 0; k < SUB; ++k) {
        const int64_t g = (int64_t)t.place * p.G + (pc * V + k * (V / SUB)) / p.per;
        mean[k] = __ldg(&p.mean[g]);
        rstd[k] = __ldg(&p.rstd[g]);
      }
#pragma unroll
      for (int i = 0; i < P; ++i) {
        a[i] = b[i] = both(0.f);
        scale[i] = __fmul2_rn(of_pair<V, SUB>(rstd, i), pair_at<V>(p.gamma, pc * V + 2 * i, 1.f));
        beta[i] = pair_at<V>(p.beta, pc * V + 2 * i, 0.f);
      }
      walk<2>(rows_of(p, at, t.hi - t.lo), [&](int j) { return Pair<T, V>{load_piece<T, V>(x + j * step), load_piece<T, V>(dy + j * dy_step)}; },
              [&](int, const Pair<T, V>& q) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
          const float2 d = less(pair_of<T, V>(q.x, i), of_pair<V, SUB>(mean, i));
          const float2 dz = through<ACT>(pair_of<T, V>(q.dy, i), __ffma2_rn(d, scale[i], beta[i]));
          a[i] = __fadd2_rn(a[i], dz);
          b[i] = __ffma2_rn(dz, d, b[i]);
        }
      });
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const int c = at.ty * W + at.tx * V + 2 * i;
        b[i] = __fmul2_rn(b[i], of_pair<V, SUB>(rstd, i));
        s_a[c] = a[i].x;
        s_b[c] = b[i].x;
        if (V > 1) {
          s_a[c + 1] = a[i].y;
          s_b[c + 1] = b[i].y;
        }
      }
    }
    __syncthreads();
    const int c0 = (pc - at.tx) * V;
    per_channel(W, [&](int c, int y0, int share) {
      const bool live = c < W && c0 + c < p.C;
      float a = 0.f, b = 0.f;
      if (live)
        for (int y = y0; y < at.tys; y += share) {
          a += s_a[y * W + c];
          b += s_b[y * W + c];
        }
      a = sum_over(a, share);
      b = sum_over(b, share);
      if (!live || y0) return;
      const float gamma = p.gamma ? __ldg(&p.gamma[c0 + c]) : 1.f;
      if (p.channels) {
        p.channels[(int64_t)tile * 2 * p.C + c0 + c] = a;
        p.channels[(int64_t)tile * 2 * p.C + p.C + c0 + c] = b;
      }
      c_a[c0 + c] = gamma * a;
      c_b[c0 + c] = gamma * b;
    });
    __syncthreads();
  }
  per_group(p.G, [&](int g, int lane, int width) {
    float a = 0.f, b = 0.f;
    if (g < p.G)
      for (int c = lane; c < p.per; c += width) {
        a += c_a[g * p.per + c];
        b += c_b[g * p.per + c];
      }
    a = sum_over(a, width);
    b = sum_over(b, width);
    if (g < p.G && lane == 0) p.part[(int64_t)tile * p.G + g] = make_float2(a, b);
  });
}

template <typename T, int V, int ACT, int SUB, typename R>
__device__ __forceinline__ void tile_grad_apply(const Params& p, const Place& at, const Tile& t, R&& ready) {
  const bool ok = ready();   // (asking for more before that costs registers, and with SiLU 6 %)
  if (at.ty >= at.tys) return;
  const int64_t step = (int64_t)at.tys * p.x_ld, dy_step = (int64_t)at.tys * p.dy_ld, out_step = (int64_t)at.tys * p.C;
  for (int pc = at.tx; pc < at.pieces; pc += at.txs) {
    const T* const x = reinterpret_cast<const T*>(p.x) + (int64_t)(t.lo + at.ty) * p.x_ld + pc * V;
    const T* const dy = reinterpret_cast<const T*>(p.dy) + (int64_t)(t.lo + at.ty) * p.dy_ld + pc * V;
    T* const dx = reinterpret_cast<T*>(p.out) + (int64_t)(t.lo + at.ty) * p.C + pc * V;
    constexpr int P = (V + 1) / 2;
    float mean[SUB], rstd[SUB], a[SUB], b[SUB];   // (the sums' negatives over std, over its square)
    float2 scale[P], beta[P];
#pragma unroll
    for (int k = 0; k < SUB; ++k) {
      const int g = (pc * V + k * (V / SUB)) / p.per;
      mean[k] = __ldg(&p.mean[(int64_t)t.place * p.G + g]);
      rstd[k] = __ldg(&p.rstd[(int64_t)t.place * p.G + g]);
      const float2 v = ok ? __ldcg(&p.whole[(int64_t)t.scene * p.G + g]) : make_float2(__int_as_float(0x7FC00000), 0.f);
      a[k] = -rstd[k] * v.x;
      b[k] = -rstd[k] * (rstd[k] * v.y);
    }
#pragma unroll
    for (int i = 0; i < P; ++i) {
      scale[i] = __fmul2_rn(of_pair<V, SUB>(rstd, i), pair_at<V>(p.gamma, pc * V + 2 * i, 1.f));
      beta[i] = pair_at<V>(p.beta, pc * V + 2 * i, 0.f);
    }
    walk<2>(rows_of(p, at, t.hi - t.lo), [&](int j) { return Pair<T, V>{load_last<T, V>(x + j * step), load_last<T, V>(dy + j * dy_step)}; },
            [&](int j, const Pair<T, V>& q) {
      float2 o[P];
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const float2 d = less(pair_of<T, V>(q.x, i), of_pair<V, SUB>(mean, i));
        const float2 dz = through<ACT>(pair_of<T, V>(q.dy, i), __ffma2_rn(d, scale[i], beta[i]));
        o[i] = __ffma2_rn(d, of_pair<V, SUB>(b, i), __ffma2_rn(scale[i], dz, of_pair<V, SUB>(a, i)));
      }
      store_piece<T, V>(dx + j * out_step, rounded<T, V>(o));
    });
  }
}

// Sums of eight channels over all tiles, 32 tiles side by side, in double.
constexpr int JOINED = 8;
__device__ __forceinline__ void join_channels(const Params& p, int c0, bool ok, float* smem) {
  constexpr int SIDE = THREADS / JOINED;
  double (*const s)[JOINED + 1] = reinterpret_cast<double(*)[JOINED + 1]>(smem);
  const int x = threadIdx.x % JOINED, y = threadIdx.x / JOINED, n = 2 * p.C, c = c0 + x;
  double v = 0;
  if (c < n) {
#pragma unroll 8
    for (int i = y; i < p.tiles; i += SIDE) v += (double)__ldcg(&p.channels[(int64_t)i * n + c]);
  }
  s[y][x] = v;
  __syncthreads();
  if (y || c >= n) return;
  for (int k = 1; k < SIDE; ++k) v += s[k][x];
  if (p.add) v += (double)p.sums[c];
  p.sums[c] = ok ? (float)v : __int_as_float(0x7FC00000);
}

// Item k of a launch: the first look at a tile, the second one, or (backward) sums of channels behind all of them.
struct Item { int kind, at; };
__device__ __forceinline__ Item item_of(const Params& p, int k, bool apply) {
  if (!apply) return k < p.tiles ? Item{0, k} : Item{2, k - p.tiles};
  if (k < p.lag) return {0, k};
  const int j = k - p.lag, both = 2 * (p.tiles - p.lag);
  if (j < both) return {j & 1, (j & 1 ? 0 : p.lag) + j / 2};
  return j - both < p.lag ? Item{1, p.tiles - p.lag + j - both} : Item{2, j - both - p.lag};
}

template <typename T, int V, int ACT, int SUB, bool BACK>
__global__ void __launch_bounds__(THREADS, BACK ? BLOCKS_BACKWARD : BLOCKS_FORWARD) group_norm_kernel(const __grid_constant__ Scenes scenes, const __grid_constant__ Params p) {
  extern __shared__ __align__(16) float smem[];
  __shared__ int s_item, s_last, s_ok, s_failed;
  const bool apply = p.out != nullptr;
  const Place at(p.C, V);
  if (threadIdx.x == 0) {
    s_item = atomicAdd(&p.sync->ticket, 1);
    s_failed = *(volatile int32_t*)p.dev_status == (int)WCN_ERR_WAIT_EXPIRED;   // (an earlier launch gave up: no results)
  }
  __syncthreads();
  for (;;) {
    const int k = s_item;
    if (k >= p.items) break;
    int next = 0;
    if (threadIdx.x == 0) next = atomicAdd(&p.sync->ticket, 1);   // (arrives while this item is worked on)
    const Item it = item_of(p, k, apply);
    if (it.kind == 2) {
      if (threadIdx.x == 0) s_ok = !s_failed && wait_for(&p.sync->scenes, scenes.count, p.dev_status);
      __syncthreads();
      join_channels(p, it.at * JOINED, s_ok, smem);
    } else {
      const Tile t = find_tile(scenes, it.at, p.rows);
      if (it.kind == 0) {
        if constexpr (BACK) tile_grad_sums<T, V, ACT, SUB>(p, at, t, it.at, smem);
        else tile_stats<T, V>(p, at, t, it.at, smem);
        __syncthreads();
        if (threadIdx.x == 0) {
          __threadfence();   // (of what the block has written)
          s_last = atomicAdd(&p.sync->tiles[t.scene], 1) == t.last - t.first - 1;
        }
        __syncthreads();
        if (s_last) {
          __threadfence();
          const int n = scenes.row0[t.scene + 1] - scenes.row0[t.scene];
          if constexpr (BACK) join_grad_sums(p, t, n);
          else join_stats<T, V>(p, t, n);
          __syncthreads();
          if (threadIdx.x == 0) {
            __threadfence();
            store_release(&p.sync->flag[t.scene], 1);
            atomicAdd(&p.sync->scenes, 1);
          }
        }
      } else {
        auto ready = [&]() -> bool {
          if (threadIdx.x == 0) s_ok = !s_failed && wait_for(&p.sync->flag[t.scene], 1, p.dev_status);
          __syncthreads();
          return s_ok;
        };
        if constexpr (BACK) tile_grad_apply<T, V, ACT, SUB>(p, at, t, ready);
        else tile_apply<T, V, ACT, SUB>(p, at, t, ready);
      }
    }
    __syncthreads();
    if (threadIdx.x == 0) s_item = next;
    __syncthreads();
  }
  // the last block leaves everything zero
  if (threadIdx.x == 0) {
    __threadfence();
    s_last = atomicAdd(&p.sync->done, 1) == (int)gridDim.x - 1;
  }
  __syncthreads();
  if (!s_last) return;
  for (int i = threadIdx.x; i < (int)(sizeof(Sync) / 4); i += THREADS) reinterpret_cast<int*>(p.sync)[i] = 0;
}

// ------------------------------------------------------------------ launches

struct Plan {
  int vec;       // elements of a piece
  int tys;       // rows of a tile side by side
};

Plan plan(int C, int elem, bool aligned) {
  Plan q;
  q.vec = aligned && C % (16 / elem) == 0 ? 16 / elem : 1;
  const int pieces = C / q.vec;
  q.tys = THREADS / (pieces < THREADS ? pieces : THREADS);
  return q;
}

size_t sums_smem(int C, int vec) {
  const int pieces = C / vec, txs = pieces < THREADS ? pieces : THREADS, tys = THREADS / txs;
  const size_t bytes = ((size_t)2 * tys * txs * vec + 2 * C) * sizeof(float), channels = THREADS / JOINED * (JOINED + 1) * sizeof(double);
  return bytes > channels ? bytes : channels;
}

// Scenes [i, j) of a launch.
struct Part { int64_t i, j; int rows, tiles, most; };   // rows of a tile; tiles of all scenes and of the longest one

// f(part) for each launch.  Tiles of up to 64 rows a thread (32 backward, where there are two numbers for each), of such a size
// that the blocks have whole rounds of them (8 x 150 000 x 96 fp16: seven rounds of 64 rows or eight of 49 for both looks).
template <typename F> int in_launches(const int64_t* offsets, int64_t scenes, bool back, int tys, F&& f) {
  for (int64_t i = 0; i < scenes;) {
    Part q = {i, i, 0, 0, 0};
    int count = 0;   // scenes with rows
    for (; q.j < scenes && count < SCENES; ++q.j) count += offsets[q.j + 1] > offsets[q.j];
    const int64_t n = offsets[q.j] - offsets[i], blocks = (back ? BLOCKS_BACKWARD : BLOCKS_FORWARD) * wcn_num_sms(), side = tys * blocks;
    const int64_t most = back ? 32 : 64, least = 4, rounds = (n + side * most - 1) / (side * most);
    int64_t per = rounds ? (n + side * rounds - 1) / (side * rounds) : least;
    if (per < least) per = least;
    for (int tries = 0;; ++tries, ++per) {
      q.rows = (int)per * tys;
      q.tiles = q.most = 0;
      for (int64_t k = i; k < q.j; ++k) {
        const int tiles = (int)((offsets[k + 1] - offsets[k] + q.rows - 1) / q.rows);
        q.tiles += tiles;
        if (tiles > q.most) q.most = tiles;
      }
      if (q.tiles <= rounds * blocks || tries == 3 || count > 16) break;   // (the scenes' last tiles are smaller ones)
    }
    i = q.j;
    const int rc = q.tiles ? f(q) : WCN_OK;
    if (rc != WCN_OK) return rc;
  }
  return WCN_OK;
}

template <typename T, int V, int ACT, int SUB, bool BACK> int all_launches(Params p, const int64_t* offsets, int64_t scenes, cudaStream_t st) {
  const Params base = p;
  const size_t smem = sums_smem(p.C, V);
  const int pieces = p.C / V, tys = THREADS / (pieces < THREADS ? pieces : THREADS);
  auto kern = group_norm_kernel<T, V, ACT, SUB, BACK>;
  if (smem > 40 * 1024 && cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) {
    (void)cudaGetLastError();
    return WCN_ERR_INITIALIZATION;
  }
  return in_launches(offsets, scenes, BACK, tys, [&](const Part& q) {
    const int64_t r = offsets[q.i];
    Scenes s;
    s.count = 0;
    int at = 0;   // (mean and rstd are those of all scenes, also of the empty ones, which a launch leaves out)
    for (int64_t k = q.i; k < q.j; ++k) {
      if (offsets[k + 1] == offsets[k]) continue;
      s.scene[s.count] = (int)(k - q.i);
      s.row0[s.count] = (int)(offsets[k] - r);
      s.tile0[s.count++] = at;
      at += (int)((offsets[k + 1] - offsets[k] + q.rows - 1) / q.rows);
    }
    s.row0[s.count] = (int)(offsets[q.j] - r);
    s.tile0[s.count] = at;
    const int grid_most = (BACK ? BLOCKS_BACKWARD : BLOCKS_FORWARD) * wcn_num_sms();
    p.rows = q.rows;
    p.each = q.rows / tys;
    p.tiles = q.tiles;
    const int lag = q.most + grid_most;   // (what was claimed a grid of tiles ago is done: blocks hardly ever wait)
    p.lag = lag < q.tiles ? lag : q.tiles;
    p.x = reinterpret_cast<const T*>(base.x) + r * p.x_ld;
    if (BACK) p.dy = reinterpret_cast<const T*>(base.dy) + r * p.dy_ld;
    p.out = base.out ? reinterpret_cast<T*>(base.out) + r * p.C : nullptr;
    p.mean = base.mean ? base.mean + q.i * p.G : nullptr;
    p.rstd = base.rstd ? base.rstd + q.i * p.G : nullptr;
    p.items = (p.out ? 2 : 1) * q.tiles + (p.sums ? (2 * p.C + JOINED - 1) / JOINED : 0);
    kern<<<p.items < grid_most ? p.items : grid_most, THREADS, smem, st>>>(s, p);
    ++wcn_launched;
    p.add = 1;
    return cudaGetLastError() == cudaSuccess ? WCN_OK : WCN_ERR_EXECUTION;
  });
}

template <typename T, int V, int ACT, int SUB> int by_way(bool back, const Params& p, const int64_t* offsets, int64_t scenes, cudaStream_t st) {
  return back ? all_launches<T, V, ACT, SUB, true>(p, offsets, scenes, st) : all_launches<T, V, ACT, SUB, false>(p, offsets, scenes, st);
}
template <typename T, int V, int SUB> int by_act(int act, bool back, const Params& p, const int64_t* offsets, int64_t scenes, cudaStream_t st) {
  switch (act) {
    case NONE: return by_way<T, V, NONE, SUB>(back, p, offsets, scenes, st);
    case RELU: return by_way<T, V, RELU, SUB>(back, p, offsets, scenes, st);
    case SILU: return by_way<T, V, SILU, SUB>(back, p, offsets, scenes, st);
    default: return by_way<T, V, GELU, SUB>(back, p, offsets, scenes, st);
  }
}

template <typename T> int by_vec(int vec, int act, bool back, const Params& p, const int64_t* offsets, int64_t scenes, cudaStream_t st) {
  constexpr int V = 16 / (int)sizeof(T);
  if (vec == 1) return by_act<T, 1, 1>(act, back, p, offsets, scenes, st);
  if (p.per % V == 0) return by_act<T, V, 1>(act, back, p, offsets, scenes, st);
  if (p.per % (V / 2) == 0) return by_act<T, V, 2>(act, back, p, offsets, scenes, st);
  return by_act<T, V, V>(act, back, p, offsets, scenes, st);
}

int by_dtype(int dtype, int vec, int act, bool back, const Params& p, const int64_t* offsets, int64_t scenes, cudaStream_t st) {
  if (dtype == WCN_F32) return by_vec<float>(vec, act, back, p, offsets, scenes, st);
  if (dtype == WCN_F16) return by_vec<__half>(vec, act, back, p, offsets, scenes, st);
  return by_vec<__nv_bfloat16>(vec, act, back, p, offsets, scenes, st);
}

bool norm_ok(int64_t scenes, const int64_t* offsets, int C, int G, int dtype) {
  if (dtype < WCN_F32 || dtype > WCN_BF16 || scenes < 0 || !offsets || C <= 0 || C > MAX_C || G <= 0 || C % G) return false;
  if (offsets[0] != 0 || offsets[scenes] >= 0x7FFF0000ll) return false;
  for (int64_t i = 0; i < scenes; ++i)
    if (offsets[i + 1] < offsets[i]) return false;
  return true;
}

bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool in_pieces(const void* p, int64_t ld, int elem) { return on16(p) && ld * elem % 16 == 0; }

float from_bits(uint32_t b) {
  float f;
  memcpy(&f, &b, sizeof f);
  return f;
}

// Where a launch keeps what its tiles leave: sums of the groups, of whole scenes, of the channels (backward).
struct Room { int64_t whole, channels, bytes; };
Room room(const int64_t* offsets, int64_t scenes, int C, int G, bool back, bool channels, int tys) {
  int64_t most = 0;
  in_launches(offsets, scenes, back, tys, [&](const Part& q) {
    if (q.tiles > most) most = q.tiles;
    return (int)WCN_OK;
  });
  Room r;
  r.whole = (most * G * (int64_t)sizeof(float2) + 255) / 256 * 256;
  r.channels = r.whole + ((scenes < SCENES ? scenes : SCENES) * G * (int64_t)sizeof(float2) + 255) / 256 * 256;
  r.bytes = r.channels + (channels ? most * 2 * C * 4 : 0);
  return r;
}

}  // namespace

extern "C" int wcn_group_norm_workspace_bytes(const int64_t* offsets, int64_t scenes, int32_t channels, int32_t groups, int dtype,
                                              int backward, int64_t* bytes) {
  if (!bytes || !norm_ok(scenes, offsets, channels, groups, dtype)) return WCN_ERR_INVALID_PARAMETERS;
  int64_t most = 0;
  for (int v = 0; v < 2; ++v) {   // (whatever the rows' alignment will be)
    const Room r = room(offsets, scenes, channels, groups, backward, backward, plan(channels, wcn_dtype_size(dtype), v).tys);
    if (r.bytes > most) most = r.bytes;
  }
  *bytes = most;
  return WCN_OK;
}

extern "C" int wcn_group_norm_sync_bytes(int64_t* bytes) {
  if (!bytes) return WCN_ERR_INVALID_PARAMETERS;
  *bytes = sizeof(Sync);
  return WCN_OK;
}

extern "C" int wcn_group_norm(const void* x, int64_t x_ld, const int64_t* offsets, int64_t scenes, int32_t channels, int32_t groups,
                              int dtype, const float* gamma, const float* beta, uint32_t eps_bits, int act, void* y, float* mean,
                              float* rstd, void* workspace, int64_t workspace_bytes, void* sync, int32_t* dev_status, void* stream) {
  wcn_launched = 0;
  if (!norm_ok(scenes, offsets, channels, groups, dtype) || act < NONE || act > GELU || x_ld < channels || !mean != !rstd)
    return WCN_ERR_INVALID_PARAMETERS;
  if (!offsets[scenes]) return WCN_OK;
  if (!x || !y || !workspace || !on16(workspace) || !sync || !dev_status) return WCN_ERR_INVALID_PARAMETERS;
  const int elem = wcn_dtype_size(dtype);
  const Plan q = plan(channels, elem, in_pieces(x, x_ld, elem) && in_pieces(y, channels, elem));
  const Room r = room(offsets, scenes, channels, groups, false, false, q.tys);
  if (r.bytes > workspace_bytes) return WCN_ERR_SCRATCH_TOO_SMALL;
  Params p = {};
  p.x = x; p.out = y; p.gamma = gamma; p.beta = beta; p.mean = mean; p.rstd = rstd;
  p.part = (float2*)workspace; p.whole = (float2*)((char*)workspace + r.whole); p.sync = (Sync*)sync; p.dev_status = dev_status;
  p.x_ld = x_ld; p.C = channels; p.G = groups; p.per = channels / groups; p.eps = from_bits(eps_bits);
  return by_dtype(dtype, q.vec, act, false, p, offsets, scenes, wcn_stream(stream));
}

extern "C" int wcn_group_norm_backward(const void* x, int64_t x_ld, const void* dy, int64_t dy_ld, const int64_t* offsets,
                                       int64_t scenes, int32_t channels, int32_t groups, int dtype, const float* gamma,
                                       const float* beta, const float* mean, const float* rstd, int act, void* dx, float* sums,
                                       void* workspace, int64_t workspace_bytes, void* sync, int32_t* dev_status, void* stream) {
  wcn_launched = 0;
  if (!norm_ok(scenes, offsets, channels, groups, dtype) || act < NONE || act > GELU || x_ld < channels || dy_ld < channels)
    return WCN_ERR_INVALID_PARAMETERS;
  cudaStream_t st = wcn_stream(stream);
  if (!offsets[scenes]) return !sums || cudaMemsetAsync(sums, 0, (size_t)2 * channels * 4, st) == cudaSuccess ? WCN_OK : WCN_ERR_EXECUTION;
  if (!x || !dy || !mean || !rstd || !workspace || !on16(workspace) || !sync || !dev_status) return WCN_ERR_INVALID_PARAMETERS;
  const int elem = wcn_dtype_size(dtype);
  const Plan q = plan(channels, elem, in_pieces(x, x_ld, elem) && in_pieces(dy, dy_ld, elem) && in_pieces(dx, channels, elem));
  const Room r = room(offsets, scenes, channels, groups, true, sums, q.tys);
  if (r.bytes > workspace_bytes) return WCN_ERR_SCRATCH_TOO_SMALL;
  Params p = {};
  p.x = x; p.dy = dy; p.out = dx; p.gamma = gamma; p.beta = beta; p.mean = const_cast<float*>(mean); p.rstd = const_cast<float*>(rstd);
  p.part = (float2*)workspace; p.whole = (float2*)((char*)workspace + r.whole); p.sync = (Sync*)sync; p.dev_status = dev_status;
  p.channels = sums ? (float*)((char*)workspace + r.channels) : nullptr;
  p.sums = sums;
  p.x_ld = x_ld; p.dy_ld = dy_ld; p.C = channels; p.G = groups; p.per = channels / groups;
  if (!dx && !sums) return WCN_OK;
  return by_dtype(dtype, q.vec, act, true, p, offsets, scenes, st);
}
