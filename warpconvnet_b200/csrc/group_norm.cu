// Group normalisation of [N, C] rows per scene, with the activation behind it:
//     mean, var of (rows of the scene) x (channels of the group);  xhat = (x - mean) / sqrt(var + eps)
//     y = act(gamma xhat + beta)                                   act: none, ReLU, SiLU, GELU
// and its gradients, with dz = dy act'(gamma xhat + beta) and M values in a (scene, group):
//     dbeta = sum dz,  dgamma = sum dz xhat,  dx = (gamma dz - sum(gamma dz) / M - xhat sum(gamma dz xhat) / M) / std.
//
// Bound by HBM where the rows are larger than L2, by L2 and latency below.  Each direction looks at the rows twice, first for
// sums, then to write the result.  The scenes are worked through in groups of up to GROUP_BYTES, a launch per look, so that the
// second one finds the rows in L2: HBM sees them once (scenes larger than that twice).  A thread owns 16 bytes of channels and
// walks the rows of a tile of its scene; a tile leaves one mean and one sum of squared distances from it per group (backward:
// two sums), and each block of the second look puts the tiles of its scene together itself, in their order and in double: no
// block waits for another and the bits are the same on every run.
// Variances are never differences of large numbers: eight rows of a thread at a time have a mean of their own, and means are
// put together by their differences.  A row far from all others or a mean that is large against the spread costs no precision.
#include <string.h>

#include "wcn_common.cuh"

namespace {

constexpr int THREADS = 256;
constexpr int ROWS = 8;                          // rows of a thread at a time
constexpr int FEW = 24, MANY = 1000;             // scenes of a launch: 0.3 and 12 KB of parameters
constexpr int MAX_C = 4096;
constexpr int64_t GROUP_BYTES = 48ll << 20;

enum Act { NONE = 0, RELU = 1, SILU = 2, GELU = 3 };

template <int M> struct Scenes {
  int count;
  int row0[M + 1];    // first row, from the launch's first row on
  int tile0[M + 1];   // first tile
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
  float* channels;        // [tiles][2][C] backward: sum dz, sum dz xhat
  int64_t x_ld, dy_ld;
  int C, G, per;          // per: channels of a group
  int rows;               // rows of a tile
  float eps;
};

template <typename T, int V> struct Piece { T v[V]; };
template <typename T, int V> __device__ __forceinline__ Piece<T, V> load_piece(const T* p) {
  Piece<T, V> q;
  if constexpr (V * sizeof(T) == 16) *reinterpret_cast<uint4*>(q.v) = __ldg(reinterpret_cast<const uint4*>(p));
  else
    for (int i = 0; i < V; ++i) q.v[i] = p[i];
  return q;
}
template <typename T, int V> __device__ __forceinline__ void store_piece(T* p, const Piece<T, V>& q) {
  if constexpr (V * sizeof(T) == 16) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(q.v);
  else
    for (int i = 0; i < V; ++i) p[i] = q.v[i];
}

template <int ACT> __device__ __forceinline__ float activate(float z) {
  if (ACT == RELU) return z > 0.f || z != z ? z : 0.f;
  if (ACT == SILU) return __fdividef(z, 1.f + __expf(-z));
  if (ACT == GELU) return z * 0.5f * (1.f + erff(z * 0.70710678118654752f));
  return z;
}
// dy act'(z)
template <int ACT> __device__ __forceinline__ float through(float dy, float z) {
  if (ACT == RELU) return z > 0.f || z != z ? dy : 0.f;
  if (ACT == SILU) {
    const float p = __fdividef(1.f, 1.f + __expf(-z));
    return dy * (p * fmaf(z, 1.f - p, 1.f));
  }
  if (ACT == GELU) return dy * (0.5f * (1.f + erff(z * 0.70710678118654752f)) + z * 0.3989422804014327f * __expf(-0.5f * z * z));
  return dy;
}

// The scene and the rows of a block's tile.
struct Tile { int scene, lo, hi, first, last; };   // first, last + 1: tiles of the scene
template <int M> __device__ __forceinline__ Tile find_tile(const Scenes<M>& s, int rows) {
  int at = 0;
  for (int hi = s.count; hi - at > 1;) {
    const int mid = (at + hi) / 2;
    if (s.tile0[mid] <= (int)blockIdx.x) at = mid; else hi = mid;
  }
  Tile t{at, 0, 0, s.tile0[at], s.tile0[at + 1]};
  t.lo = s.row0[at] + ((int)blockIdx.x - t.first) * rows;
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

template <typename T, int V, int M>
__global__ void __launch_bounds__(THREADS) group_stats_kernel(const __grid_constant__ Scenes<M> scenes, const __grid_constant__ Params p) {
  extern __shared__ __align__(16) float smem[];
  const Place at(p.C, V);
  const int W = at.txs * V;                       // channels side by side
  float* const s_mean = smem;                     // [tys][W]
  float* const s_m2 = smem + at.tys * W;          // [tys][W]
  float* const c_mean = s_m2 + at.tys * W;        // [C]
  float* const c_m2 = c_mean + p.C;               // [C]
  const Tile t = find_tile(scenes, p.rows);
  const int n_tile = t.hi - t.lo;
  const T* const x = reinterpret_cast<const T*>(p.x);
  for (int pc = at.tx; pc - at.tx < at.pieces; pc += at.txs) {
    const bool live = at.ty < at.tys && pc < at.pieces;
    float mean[V], m2[V];
#pragma unroll
    for (int i = 0; i < V; ++i) mean[i] = m2[i] = 0.f;
    if (live) {
      int n = 0;
      for (int r = t.lo + at.ty; r < t.hi; r += ROWS * at.tys) {
        Piece<T, V> q[ROWS];
        int k = 0;
#pragma unroll
        for (int u = 0; u < ROWS; ++u)
          if (r + u * at.tys < t.hi) {
            q[u] = load_piece<T, V>(x + (int64_t)(r + u * at.tys) * p.x_ld + pc * V);
            k = u + 1;
          }
        const float inv = 1.f / (float)k, share = (float)k / (float)(n + k);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float sum = 0.f, d2 = 0.f;
#pragma unroll
          for (int u = 0; u < ROWS; ++u) sum += u < k ? wcn_to_float<T>(q[u].v[i]) : 0.f;
          const float mb = sum * inv;
#pragma unroll
          for (int u = 0; u < ROWS; ++u) {
            const float d = u < k ? wcn_to_float<T>(q[u].v[i]) - mb : 0.f;
            d2 = fmaf(d, d, d2);
          }
          const float delta = mb - mean[i];
          mean[i] = fmaf(delta, share, mean[i]);
          m2[i] += d2 + delta * delta * (share * (float)n);
        }
        n += k;
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        s_mean[at.ty * W + at.tx * V + i] = mean[i];
        s_m2[at.ty * W + at.tx * V + i] = m2[i];
      }
    }
    __syncthreads();
    const int c0 = (pc - at.tx) * V;
    for (int c = threadIdx.x; c < W && c0 + c < p.C; c += THREADS) {
      float sum = 0.f, m2c = 0.f;
      // rows ty, ty + tys, ... of the tile
      for (int y = 0; y < at.tys; ++y) sum = fmaf(s_mean[y * W + c], (float)((n_tile - y + at.tys - 1) / at.tys), sum);
      const float m = sum / (float)n_tile;
      for (int y = 0; y < at.tys; ++y) {
        const float d = s_mean[y * W + c] - m;
        m2c += s_m2[y * W + c] + d * d * (float)((n_tile - y + at.tys - 1) / at.tys);
      }
      c_mean[c0 + c] = m;
      c_m2[c0 + c] = m2c;
    }
    __syncthreads();
  }
  // a warp puts the channels of a group together
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int g = warp; g < p.G; g += THREADS / 32) {
    float sum = 0.f, m2g = 0.f;
    for (int c = lane; c < p.per; c += 32) sum += c_mean[g * p.per + c];
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    const float m = sum / (float)p.per;
    for (int c = lane; c < p.per; c += 32) {
      const float d = c_mean[g * p.per + c] - m;
      m2g += c_m2[g * p.per + c] + d * d * (float)n_tile;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) m2g += __shfl_xor_sync(0xFFFFFFFFu, m2g, o);
    if (lane == 0) p.part[(int64_t)blockIdx.x * p.G + g] = make_float2(m, m2g);
  }
}

// What each group's tiles come to together, by as many threads a group as there are, lanes of one warp.
template <typename F> __device__ __forceinline__ void per_group(int G, F&& f) {
  int width = 32;
  while (width > 1 && width * G > THREADS) width >>= 1;
  for (int g0 = 0; g0 < G; g0 += THREADS / width) f(g0 + (int)threadIdx.x / width, (int)threadIdx.x % width, width);
}
__device__ __forceinline__ double sum_over(double v, int width) {
  for (int o = width >> 1; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

template <typename T, int V, int ACT, int M>
__global__ void __launch_bounds__(THREADS) group_apply_kernel(const __grid_constant__ Scenes<M> scenes, const __grid_constant__ Params p) {
  extern __shared__ __align__(16) float smem[];
  float* const s_mean = smem;       // [G]
  float* const s_rstd = smem + p.G;
  const Place at(p.C, V);
  const Tile t = find_tile(scenes, p.rows);
  const int n_scene = scenes.row0[t.scene + 1] - scenes.row0[t.scene];
  const int n_last = n_scene - (t.last - t.first - 1) * p.rows;
  per_group(p.G, [&](int g, int lane, int width) {
    double sum = 0, m2 = 0;
    const bool live = g < p.G;
    if (live)
      for (int i = t.first + lane; i < t.last; i += width)
        sum += (double)__ldg(&p.part[(int64_t)i * p.G + g]).x * (i == t.last - 1 ? n_last : p.rows);
    const double mean = sum_over(sum, width) / n_scene;
    if (live)
      for (int i = t.first + lane; i < t.last; i += width) {
        const float2 v = __ldg(&p.part[(int64_t)i * p.G + g]);
        const double d = (double)v.x - mean;
        m2 += (double)v.y + d * d * ((double)(i == t.last - 1 ? n_last : p.rows) * p.per);
      }
    m2 = sum_over(m2, width);
    if (live && lane == 0) {
      const float rstd = (float)(1.0 / sqrt(m2 / ((double)n_scene * p.per) + (double)p.eps));
      s_mean[g] = (float)mean;
      s_rstd[g] = rstd;
      if ((int)blockIdx.x == t.first && p.mean) {
        p.mean[(int64_t)t.scene * p.G + g] = (float)mean;
        p.rstd[(int64_t)t.scene * p.G + g] = rstd;
      }
    }
  });
  __syncthreads();
  if (at.ty >= at.tys) return;
  const T* const x = reinterpret_cast<const T*>(p.x);
  T* const y = reinterpret_cast<T*>(p.out);
  for (int pc = at.tx; pc < at.pieces; pc += at.txs) {
    float mean[V], scale[V], beta[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = pc * V + i, g = c / p.per;
      mean[i] = s_mean[g];
      scale[i] = s_rstd[g] * (p.gamma ? __ldg(&p.gamma[c]) : 1.f);
      beta[i] = p.beta ? __ldg(&p.beta[c]) : 0.f;
    }
    for (int r = t.lo + at.ty; r < t.hi; r += 4 * at.tys) {
      Piece<T, V> q[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (r + u * at.tys < t.hi) q[u] = load_piece<T, V>(x + (int64_t)(r + u * at.tys) * p.x_ld + pc * V);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (r + u * at.tys >= t.hi) break;
        Piece<T, V> o;
#pragma unroll
        for (int i = 0; i < V; ++i) o.v[i] = wcn_from_float<T>(activate<ACT>(fmaf(wcn_to_float<T>(q[u].v[i]) - mean[i], scale[i], beta[i])));
        store_piece<T, V>(y + (int64_t)(r + u * at.tys) * p.C + pc * V, o);
      }
    }
  }
}

template <typename T, int V, int ACT, int M>
__global__ void __launch_bounds__(THREADS) group_grad_sums_kernel(const __grid_constant__ Scenes<M> scenes, const __grid_constant__ Params p) {
  extern __shared__ __align__(16) float smem[];
  const Place at(p.C, V);
  const int W = at.txs * V;
  float* const s_a = smem;                    // [tys][W]
  float* const s_b = smem + at.tys * W;       // [tys][W]
  float* const c_a = s_b + at.tys * W;        // [C] gamma dz
  float* const c_b = c_a + p.C;               // [C] gamma dz xhat
  const Tile t = find_tile(scenes, p.rows);
  const T *const x = reinterpret_cast<const T*>(p.x), *const dy = reinterpret_cast<const T*>(p.dy);
  for (int pc = at.tx; pc - at.tx < at.pieces; pc += at.txs) {
    const bool live = at.ty < at.tys && pc < at.pieces;
    if (live) {
      float a[V], b[V], mean[V], rstd[V], gamma[V], beta[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int c = pc * V + i;
        const int64_t g = (int64_t)t.scene * p.G + c / p.per;
        a[i] = b[i] = 0.f;
        mean[i] = __ldg(&p.mean[g]);
        rstd[i] = __ldg(&p.rstd[g]);
        gamma[i] = p.gamma ? __ldg(&p.gamma[c]) : 1.f;
        beta[i] = p.beta ? __ldg(&p.beta[c]) : 0.f;
      }
      for (int r = t.lo + at.ty; r < t.hi; r += 4 * at.tys) {
        Piece<T, V> q[4], d[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (r + u * at.tys < t.hi) {
            q[u] = load_piece<T, V>(x + (int64_t)(r + u * at.tys) * p.x_ld + pc * V);
            d[u] = load_piece<T, V>(dy + (int64_t)(r + u * at.tys) * p.dy_ld + pc * V);
          }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (r + u * at.tys >= t.hi) break;
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float xhat = (wcn_to_float<T>(q[u].v[i]) - mean[i]) * rstd[i];
            const float dz = through<ACT>(wcn_to_float<T>(d[u].v[i]), fmaf(xhat, gamma[i], beta[i]));
            a[i] += dz;
            b[i] = fmaf(dz, xhat, b[i]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        s_a[at.ty * W + at.tx * V + i] = a[i];
        s_b[at.ty * W + at.tx * V + i] = b[i];
      }
    }
    __syncthreads();
    const int c0 = (pc - at.tx) * V;
    for (int c = threadIdx.x; c < W && c0 + c < p.C; c += THREADS) {
      float a = 0.f, b = 0.f;
      for (int y = 0; y < at.tys; ++y) {
        a += s_a[y * W + c];
        b += s_b[y * W + c];
      }
      const float gamma = p.gamma ? __ldg(&p.gamma[c0 + c]) : 1.f;
      if (p.channels) {
        p.channels[(int64_t)blockIdx.x * 2 * p.C + c0 + c] = a;
        p.channels[(int64_t)blockIdx.x * 2 * p.C + p.C + c0 + c] = b;
      }
      c_a[c0 + c] = gamma * a;
      c_b[c0 + c] = gamma * b;
    }
    __syncthreads();
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int g = warp; g < p.G; g += THREADS / 32) {
    float a = 0.f, b = 0.f;
    for (int c = lane; c < p.per; c += 32) {
      a += c_a[g * p.per + c];
      b += c_b[g * p.per + c];
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      a += __shfl_xor_sync(0xFFFFFFFFu, a, o);
      b += __shfl_xor_sync(0xFFFFFFFFu, b, o);
    }
    if (lane == 0) p.part[(int64_t)blockIdx.x * p.G + g] = make_float2(a, b);
  }
}

template <typename T, int V, int ACT, int M>
__global__ void __launch_bounds__(THREADS) group_grad_apply_kernel(const __grid_constant__ Scenes<M> scenes, const __grid_constant__ Params p) {
  extern __shared__ __align__(16) float smem[];
  float* const s_a = smem;          // [G]
  float* const s_b = smem + p.G;
  const Place at(p.C, V);
  const Tile t = find_tile(scenes, p.rows);
  const int n_scene = scenes.row0[t.scene + 1] - scenes.row0[t.scene];
  per_group(p.G, [&](int g, int lane, int width) {
    double a = 0, b = 0;
    if (g < p.G)
      for (int i = t.first + lane; i < t.last; i += width) {
        const float2 v = __ldg(&p.part[(int64_t)i * p.G + g]);
        a += (double)v.x;
        b += (double)v.y;
      }
    a = sum_over(a, width);
    b = sum_over(b, width);
    if (g < p.G && lane == 0) {
      const double inv = 1.0 / ((double)n_scene * p.per);
      s_a[g] = (float)(a * inv);
      s_b[g] = (float)(b * inv);
    }
  });
  __syncthreads();
  if (at.ty >= at.tys) return;
  const T *const x = reinterpret_cast<const T*>(p.x), *const dy = reinterpret_cast<const T*>(p.dy);
  T* const dx = reinterpret_cast<T*>(p.out);
  for (int pc = at.tx; pc < at.pieces; pc += at.txs) {
    float mean[V], rstd[V], gamma[V], beta[V], a[V], b[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = pc * V + i, g = c / p.per;
      mean[i] = __ldg(&p.mean[(int64_t)t.scene * p.G + g]);
      rstd[i] = __ldg(&p.rstd[(int64_t)t.scene * p.G + g]);
      gamma[i] = p.gamma ? __ldg(&p.gamma[c]) : 1.f;
      beta[i] = p.beta ? __ldg(&p.beta[c]) : 0.f;
      a[i] = s_a[g];
      b[i] = s_b[g];
    }
    for (int r = t.lo + at.ty; r < t.hi; r += 2 * at.tys) {
      Piece<T, V> q[2], d[2];
#pragma unroll
      for (int u = 0; u < 2; ++u)
        if (r + u * at.tys < t.hi) {
          q[u] = load_piece<T, V>(x + (int64_t)(r + u * at.tys) * p.x_ld + pc * V);
          d[u] = load_piece<T, V>(dy + (int64_t)(r + u * at.tys) * p.dy_ld + pc * V);
        }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (r + u * at.tys >= t.hi) break;
        Piece<T, V> o;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float xhat = (wcn_to_float<T>(q[u].v[i]) - mean[i]) * rstd[i];
          const float dz = through<ACT>(wcn_to_float<T>(d[u].v[i]), fmaf(xhat, gamma[i], beta[i]));
          o.v[i] = wcn_from_float<T>(rstd[i] * (fmaf(gamma[i], dz, -a[i]) - xhat * b[i]));
        }
        store_piece<T, V>(dx + (int64_t)(r + u * at.tys) * p.C + pc * V, o);
      }
    }
  }
}

// Sums over the tiles: 32 channels a block, eight tiles side by side, in double.
__global__ void __launch_bounds__(THREADS) group_param_grads_kernel(const float* part, int64_t tiles, int n, float* out) {
  __shared__ double s[THREADS / 32][33];
  const int lane = threadIdx.x & 31, y = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  double v = 0;
  if (c < n) {
    int64_t i = y;
    for (; i + 3 * (THREADS / 32) < tiles; i += 4 * (THREADS / 32)) {
      float q[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) q[u] = __ldg(&part[(i + u * (THREADS / 32)) * n + c]);
#pragma unroll
      for (int u = 0; u < 4; ++u) v += (double)q[u];
    }
    for (; i < tiles; i += THREADS / 32) v += (double)__ldg(&part[i * n + c]);
  }
  s[y][lane] = v;
  __syncthreads();
  if (y == 0 && c < n) {
    for (int k = 1; k < THREADS / 32; ++k) v += s[k][lane];
    out[c] = (float)v;
  }
}

// ------------------------------------------------------------------ launches

struct Plan {
  int vec;       // elements of a piece
  int rows;      // rows of a tile
};

Plan plan(int64_t n, int C, int elem, bool aligned) {
  Plan q;
  q.vec = aligned && C % (16 / elem) == 0 ? 16 / elem : 1;
  const int pieces = C / q.vec, tys = THREADS / (pieces < THREADS ? pieces : THREADS);
  // four blocks an SM, one to 64 rows a thread
  int64_t per = n / ((int64_t)tys * 4 * wcn_num_sms());
  per = per < 1 ? 1 : per > 64 ? 64 : per;
  if (per > ROWS) per = per / ROWS * ROWS;
  q.rows = (int)(per * tys);
  return q;
}

size_t sums_smem(int C, int vec) {
  const int pieces = C / vec, txs = pieces < THREADS ? pieces : THREADS, tys = THREADS / txs;
  return ((size_t)2 * tys * txs * vec + 2 * C) * sizeof(float);
}

// All launches of one direction over one group of scenes: f(scenes, tiles).
template <int M, typename F> int launch_group(const int64_t* offsets, int64_t first, int64_t last, int rows, F&& f) {
  Scenes<M> s;
  s.count = (int)(last - first);
  int tiles = 0;
  for (int64_t i = first; i <= last; ++i) {
    s.row0[i - first] = (int)(offsets[i] - offsets[first]);
    s.tile0[i - first] = tiles;
    if (i < last) tiles += (int)((offsets[i + 1] - offsets[i] + rows - 1) / rows);
  }
  if (!tiles) return WCN_OK;
  return f(s, tiles);
}

// The scenes in groups that stay in L2.
template <typename F> int in_groups(const int64_t* offsets, int64_t scenes, int64_t row_bytes, F&& f) {
  for (int64_t i = 0; i < scenes;) {
    int64_t j = i + 1;
    while (j < scenes && j - i < MANY && (offsets[j + 1] - offsets[i]) * row_bytes <= GROUP_BYTES) ++j;
    const int rc = f(i, j);
    if (rc != WCN_OK) return rc;
    i = j;
  }
  return WCN_OK;
}

template <typename T, int V, int ACT, int M> int forward_group(const Scenes<M>& s, int tiles, const Params& p, cudaStream_t st) {
  group_stats_kernel<T, V, M><<<tiles, THREADS, sums_smem(p.C, V), st>>>(s, p);
  group_apply_kernel<T, V, ACT, M><<<tiles, THREADS, (size_t)2 * p.G * sizeof(float), st>>>(s, p);
  return cudaGetLastError() == cudaSuccess ? WCN_OK : WCN_ERR_EXECUTION;
}
template <typename T, int V, int ACT, int M> int backward_group(const Scenes<M>& s, int tiles, const Params& p, cudaStream_t st) {
  group_grad_sums_kernel<T, V, ACT, M><<<tiles, THREADS, sums_smem(p.C, V), st>>>(s, p);
  if (p.out) group_grad_apply_kernel<T, V, ACT, M><<<tiles, THREADS, (size_t)2 * p.G * sizeof(float), st>>>(s, p);
  return cudaGetLastError() == cudaSuccess ? WCN_OK : WCN_ERR_EXECUTION;
}

template <typename T, int V, int ACT> int all_groups(bool back, Params p, const int64_t* offsets, int64_t scenes, cudaStream_t st) {
  const int64_t row_bytes = (int64_t)p.C * sizeof(T) * (back ? 2 : 1);
  const Params base = p;
  return in_groups(offsets, scenes, row_bytes, [&](int64_t i, int64_t j) {
    const int64_t r = offsets[i];
    p.x = reinterpret_cast<const T*>(base.x) + r * p.x_ld;
    if (back) p.dy = reinterpret_cast<const T*>(base.dy) + r * p.dy_ld;
    p.out = base.out ? reinterpret_cast<T*>(base.out) + r * p.C : nullptr;
    p.mean = base.mean ? base.mean + i * p.G : nullptr;
    p.rstd = base.rstd ? base.rstd + i * p.G : nullptr;
    auto go = [&](const auto& s, int tiles) {
      constexpr int M = sizeof(s) == sizeof(Scenes<FEW>) ? FEW : MANY;
      const int rc = back ? backward_group<T, V, ACT, M>(s, tiles, p, st) : forward_group<T, V, ACT, M>(s, tiles, p, st);
      if (back) {  // (the forward's tiles are done with once its second launch is)
        p.part += (int64_t)tiles * p.G;
        if (p.channels) p.channels += (int64_t)tiles * 2 * p.C;
      }
      return rc;
    };
    return j - i <= FEW ? launch_group<FEW>(offsets, i, j, p.rows, go) : launch_group<MANY>(offsets, i, j, p.rows, go);
  });
}

template <typename T, int V> int by_act(int act, bool back, const Params& p, const int64_t* offsets, int64_t scenes, cudaStream_t st) {
  switch (act) {
    case NONE: return all_groups<T, V, NONE>(back, p, offsets, scenes, st);
    case RELU: return all_groups<T, V, RELU>(back, p, offsets, scenes, st);
    case SILU: return all_groups<T, V, SILU>(back, p, offsets, scenes, st);
    default: return all_groups<T, V, GELU>(back, p, offsets, scenes, st);
  }
}

template <typename T> int by_vec(int vec, int act, bool back, const Params& p, const int64_t* offsets, int64_t scenes, cudaStream_t st) {
  return vec == 1 ? by_act<T, 1>(act, back, p, offsets, scenes, st) : by_act<T, 16 / (int)sizeof(T)>(act, back, p, offsets, scenes, st);
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

int64_t count_tiles(const int64_t* offsets, int64_t scenes, int rows) {
  int64_t tiles = 0;
  for (int64_t i = 0; i < scenes; ++i) tiles += (offsets[i + 1] - offsets[i] + rows - 1) / rows;
  return tiles;
}

bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool rows_on16(const void* p, int64_t ld, int elem) { return on16(p) && ld * elem % 16 == 0; }

float from_bits(uint32_t b) {
  float f;
  memcpy(&f, &b, sizeof f);
  return f;
}

// Bytes of the groups' sums, then of the channels' (backward).
int64_t part_bytes(int64_t tiles, int G) { return (tiles * G * (int64_t)sizeof(float2) + 15) / 16 * 16; }

}  // namespace

extern "C" int wcn_group_norm_workspace_bytes(const int64_t* offsets, int64_t scenes, int32_t channels, int32_t groups, int dtype,
                                              int backward, int64_t* bytes) {
  if (!bytes || !norm_ok(scenes, offsets, channels, groups, dtype)) return WCN_ERR_INVALID_PARAMETERS;
  int64_t most = 0;
  for (int v = 0; v < 2; ++v) {   // (whatever the rows' alignment will be)
    const int64_t tiles = count_tiles(offsets, scenes, plan(offsets[scenes], channels, wcn_dtype_size(dtype), v).rows);
    const int64_t need = part_bytes(tiles, groups) + (backward ? tiles * 2 * channels * 4 : 0);
    if (need > most) most = need;
  }
  *bytes = most;
  return WCN_OK;
}

extern "C" int wcn_group_norm(const void* x, int64_t x_ld, const int64_t* offsets, int64_t scenes, int32_t channels, int32_t groups,
                              int dtype, const float* gamma, const float* beta, uint32_t eps_bits, int act, void* y, float* mean,
                              float* rstd, void* workspace, int64_t workspace_bytes, void* stream) {
  if (!norm_ok(scenes, offsets, channels, groups, dtype) || act < NONE || act > GELU || x_ld < channels || !mean != !rstd)
    return WCN_ERR_INVALID_PARAMETERS;
  if (!offsets[scenes]) return WCN_OK;
  if (!x || !y || !workspace || !on16(workspace)) return WCN_ERR_INVALID_PARAMETERS;
  const int elem = wcn_dtype_size(dtype);
  const Plan q = plan(offsets[scenes], channels, elem, rows_on16(x, x_ld, elem) && rows_on16(y, channels, elem));
  if (part_bytes(count_tiles(offsets, scenes, q.rows), groups) > workspace_bytes) return WCN_ERR_SCRATCH_TOO_SMALL;
  Params p = {};
  p.x = x; p.out = y; p.gamma = gamma; p.beta = beta; p.mean = mean; p.rstd = rstd; p.part = (float2*)workspace;
  p.x_ld = x_ld; p.C = channels; p.G = groups; p.per = channels / groups; p.rows = q.rows; p.eps = from_bits(eps_bits);
  return by_dtype(dtype, q.vec, act, false, p, offsets, scenes, wcn_stream(stream));
}

extern "C" int wcn_group_norm_backward(const void* x, int64_t x_ld, const void* dy, int64_t dy_ld, const int64_t* offsets,
                                       int64_t scenes, int32_t channels, int32_t groups, int dtype, const float* gamma,
                                       const float* beta, const float* mean, const float* rstd, int act, void* dx, float* sums,
                                       void* workspace, int64_t workspace_bytes, void* stream) {
  if (!norm_ok(scenes, offsets, channels, groups, dtype) || act < NONE || act > GELU || x_ld < channels || dy_ld < channels)
    return WCN_ERR_INVALID_PARAMETERS;
  cudaStream_t st = wcn_stream(stream);
  if (!offsets[scenes]) return !sums || cudaMemsetAsync(sums, 0, (size_t)2 * channels * 4, st) == cudaSuccess ? WCN_OK : WCN_ERR_EXECUTION;
  if (!x || !dy || !mean || !rstd || !workspace || !on16(workspace)) return WCN_ERR_INVALID_PARAMETERS;
  const int elem = wcn_dtype_size(dtype);
  const Plan q = plan(offsets[scenes], channels, elem, rows_on16(x, x_ld, elem) && rows_on16(dy, dy_ld, elem) && rows_on16(dx, channels, elem));
  const int64_t tiles = count_tiles(offsets, scenes, q.rows);
  if (part_bytes(tiles, groups) + (sums ? tiles * 2 * channels * 4 : 0) > workspace_bytes) return WCN_ERR_SCRATCH_TOO_SMALL;
  Params p = {};
  p.x = x; p.dy = dy; p.out = dx; p.gamma = gamma; p.beta = beta; p.mean = const_cast<float*>(mean); p.rstd = const_cast<float*>(rstd);
  p.part = (float2*)workspace;
  p.channels = sums ? (float*)((char*)workspace + part_bytes(tiles, groups)) : nullptr;
  p.x_ld = x_ld; p.dy_ld = dy_ld; p.C = channels; p.G = groups; p.per = channels / groups; p.rows = q.rows;
  const int rc = by_dtype(dtype, q.vec, act, true, p, offsets, scenes, st);
  if (rc != WCN_OK || !sums) return rc;
  group_param_grads_kernel<<<(2 * channels + 31) / 32, THREADS, 0, st>>>(p.channels, tiles, 2 * channels, sums);
  return cudaGetLastError() == cudaSuccess ? WCN_OK : WCN_ERR_EXECUTION;
}
