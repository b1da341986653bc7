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

constexpr int THREADS = 512;
constexpr int ROWS = 8;                          // rows of a thread at a time
constexpr int SCENES = 250;                      // of a launch: 2 KB of parameters
constexpr int MAX_C = 4096;
constexpr int64_t GROUP_BYTES = 48ll << 20;

enum Act { NONE = 0, RELU = 1, SILU = 2, GELU = 3 };

struct Scenes {
  int count;
  int row0[SCENES + 1];    // first row, from the launch's first row on
  int tile0[SCENES + 1];   // first tile
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
struct Tile { int scene, lo, hi, first, last; };   // first, last: tiles of the scene
__device__ __forceinline__ Tile find_tile(const Scenes& s, int rows) {
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

template <typename T, int V>
__global__ void __launch_bounds__(THREADS, 2) group_stats_kernel(const __grid_constant__ Scenes scenes, const __grid_constant__ Params p) {
  extern __shared__ __align__(16) float smem[];
  const Place at(p.C, V);
  const int W = at.txs * V;                       // channels side by side
  float* const s_mean = smem;                     // [tys][W]
  float* const s_m2 = smem + at.tys * W;          // [tys][W]
  float* const c_mean = s_m2 + at.tys * W;        // [C]
  float* const c_m2 = c_mean + p.C;               // [C]
  const Tile t = find_tile(scenes, p.rows);
  const int n_tile = t.hi - t.lo, n_each = n_tile / at.tys, n_more = n_tile % at.tys;   // rows of a thread: one more for the first
  const T* const x = reinterpret_cast<const T*>(p.x);
  for (int pc = at.tx; pc - at.tx < at.pieces; pc += at.txs) {
    if (at.ty < at.tys && pc < at.pieces) {
      float mean[V], m2[V];
#pragma unroll
      for (int i = 0; i < V; ++i) mean[i] = m2[i] = 0.f;
      const int64_t step = (int64_t)at.tys * p.x_ld;
      const T* from = x + (int64_t)(t.lo + at.ty) * p.x_ld + pc * V;
      int n = 0;
      const int mine = n_each + (at.ty < n_more);
      for (; n + ROWS <= mine; n += ROWS, from += ROWS * step) {
        Piece<T, V> q[ROWS];
#pragma unroll
        for (int u = 0; u < ROWS; ++u) q[u] = load_piece<T, V>(from + u * step);
        const float share = (float)ROWS / (float)(n + ROWS), both = share * (float)n;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float f[ROWS], sum = 0.f, d2 = 0.f;
#pragma unroll
          for (int u = 0; u < ROWS; ++u) { f[u] = wcn_to_float<T>(q[u].v[i]); sum += f[u]; }
          const float mb = sum * (1.f / ROWS);
#pragma unroll
          for (int u = 0; u < ROWS; ++u) { const float d = f[u] - mb; d2 = fmaf(d, d, d2); }
          const float delta = mb - mean[i];
          mean[i] = fmaf(delta, share, mean[i]);
          m2[i] += fmaf(delta * delta, both, d2);
        }
      }
      for (; n < mine; ++n, from += step) {       // the last rows one by one
        const Piece<T, V> q = load_piece<T, V>(from);
        const float share = 1.f / (float)(n + 1), both = share * (float)n;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float delta = wcn_to_float<T>(q.v[i]) - mean[i];
          mean[i] = fmaf(delta, share, mean[i]);
          m2[i] = fmaf(delta * delta, both, m2[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        s_mean[at.ty * W + at.tx * V + i] = mean[i];
        s_m2[at.ty * W + at.tx * V + i] = m2[i];
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
    if (g < p.G && lane == 0) p.part[(int64_t)blockIdx.x * p.G + g] = make_float2(m, m2);
  });
}

// A piece has SUB groups side by side (V / SUB channels of one group each; V: any).
template <typename T, int V, int ACT, int SUB>
__global__ void __launch_bounds__(THREADS, 2) group_apply_kernel(const __grid_constant__ Scenes scenes, const __grid_constant__ Params p) {
  extern __shared__ __align__(16) float smem[];
  float* const s_mean = smem;       // [G]
  float* const s_rstd = smem + p.G;
  const Place at(p.C, V);
  const Tile t = find_tile(scenes, p.rows);
  const int n_scene = scenes.row0[t.scene + 1] - scenes.row0[t.scene];
  const int n_last = n_scene - (t.last - t.first - 1) * p.rows;
  per_group(p.G, [&](int g, int lane, int width) {
    // in one pass, about the first tile's mean: what the tiles' means differ by is no more than the spread
    double n = 0, d1 = 0, d2 = 0;
    float about = 0.f;
    if (g < p.G) {
      about = __ldg(&p.part[(int64_t)t.first * p.G + g]).x;
#pragma unroll 4
      for (int i = t.first + lane; i < t.last; i += width) {
        const float2 v = __ldg(&p.part[(int64_t)i * p.G + g]);
        const double k = (double)(i == t.last - 1 ? n_last : p.rows), d = (double)v.x - (double)about;
        d1 += k * d;
        d2 += (double)v.y + k * d * d * p.per;
      }
    }
    n = (double)n_scene;
    d1 = sum_over(d1, width) / n;
    d2 = sum_over(d2, width);
    if (g < p.G && lane == 0) {
      const double var = d2 / (n * p.per) - d1 * d1;
      const float mean = (float)((double)about + d1), rstd = (float)(1.0 / sqrt((var < 0 ? 0 : var) + (double)p.eps));
      s_mean[g] = mean;
      s_rstd[g] = rstd;
      if ((int)blockIdx.x == t.first && p.mean) {
        p.mean[(int64_t)t.scene * p.G + g] = mean;
        p.rstd[(int64_t)t.scene * p.G + g] = rstd;
      }
    }
  });
  __syncthreads();
  if (at.ty >= at.tys) return;
  const T* const x = reinterpret_cast<const T*>(p.x);
  T* const y = reinterpret_cast<T*>(p.out);
  for (int pc = at.tx; pc < at.pieces; pc += at.txs) {
    float mean[SUB], scale[V], beta[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = pc * V + i, g = c / p.per;
      mean[i * SUB / V] = s_mean[g];
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
        for (int i = 0; i < V; ++i) o.v[i] = wcn_from_float<T>(activate<ACT>(fmaf(wcn_to_float<T>(q[u].v[i]) - mean[i * SUB / V], scale[i], beta[i])));
        store_piece<T, V>(y + (int64_t)(r + u * at.tys) * p.C + pc * V, o);
      }
    }
  }
}

template <typename T, int V, int ACT, int SUB>
__global__ void __launch_bounds__(THREADS, 1) group_grad_sums_kernel(const __grid_constant__ Scenes scenes, const __grid_constant__ Params p) {
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
    if (at.ty < at.tys && pc < at.pieces) {
      float a[V], b[V], mean[SUB], rstd[SUB], gamma[V], beta[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int c = pc * V + i;
        const int64_t g = (int64_t)t.scene * p.G + c / p.per;
        a[i] = b[i] = 0.f;
        mean[i * SUB / V] = __ldg(&p.mean[g]);
        rstd[i * SUB / V] = __ldg(&p.rstd[g]);
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
            const float xhat = (wcn_to_float<T>(q[u].v[i]) - mean[i * SUB / V]) * rstd[i * SUB / V];
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
        p.channels[(int64_t)blockIdx.x * 2 * p.C + c0 + c] = a;
        p.channels[(int64_t)blockIdx.x * 2 * p.C + p.C + c0 + c] = b;
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
    if (g < p.G && lane == 0) p.part[(int64_t)blockIdx.x * p.G + g] = make_float2(a, b);
  });
}

template <typename T, int V, int ACT, int SUB>
__global__ void __launch_bounds__(THREADS, 1) group_grad_apply_kernel(const __grid_constant__ Scenes scenes, const __grid_constant__ Params p) {
  extern __shared__ __align__(16) float smem[];
  float* const s_a = smem;          // [G]
  float* const s_b = smem + p.G;
  const Place at(p.C, V);
  const Tile t = find_tile(scenes, p.rows);
  const int n_scene = scenes.row0[t.scene + 1] - scenes.row0[t.scene];
  per_group(p.G, [&](int g, int lane, int width) {
    double a = 0, b = 0;
    if (g < p.G)
#pragma unroll 4
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
    float mean[SUB], rstd[SUB], gamma[V], beta[V], a[SUB], b[SUB];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = pc * V + i, g = c / p.per;
      mean[i * SUB / V] = __ldg(&p.mean[(int64_t)t.scene * p.G + g]);
      rstd[i * SUB / V] = __ldg(&p.rstd[(int64_t)t.scene * p.G + g]);
      gamma[i] = p.gamma ? __ldg(&p.gamma[c]) : 1.f;
      beta[i] = p.beta ? __ldg(&p.beta[c]) : 0.f;
      a[i * SUB / V] = s_a[g];
      b[i * SUB / V] = s_b[g];
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
        Piece<T, V> o;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int k = i * SUB / V;
          const float xhat = (wcn_to_float<T>(q[u].v[i]) - mean[k]) * rstd[k];
          const float dz = through<ACT>(wcn_to_float<T>(d[u].v[i]), fmaf(xhat, gamma[i], beta[i]));
          o.v[i] = wcn_from_float<T>(rstd[k] * (fmaf(gamma[i], dz, -a[k]) - xhat * b[k]));
        }
        store_piece<T, V>(dx + (int64_t)(r + u * at.tys) * p.C + pc * V, o);
      }
    }
  }
}

// Sums over the tiles: 32 channels a block, 32 tiles side by side, in double.
__global__ void __launch_bounds__(1024) group_param_grads_kernel(const float* part, int64_t tiles, int n, float* out) {
  __shared__ double s[32][33];
  const int lane = threadIdx.x & 31, y = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  double v = 0;
  if (c < n) {
#pragma unroll 8
    for (int64_t i = y; i < tiles; i += 32) v += (double)__ldg(&part[i * n + c]);
  }
  s[y][lane] = v;
  __syncthreads();
  v = sum_over(s[lane][y], 32);   // (a warp a channel)
  if (lane == 0 && blockIdx.x * 32 + y < n) out[blockIdx.x * 32 + y] = (float)v;
}

// ------------------------------------------------------------------ launches

struct Plan {
  int vec;       // elements of a piece
  int tys;       // rows of a block side by side
};

Plan plan(int C, int elem, bool aligned) {
  Plan q;
  q.vec = aligned && C % (16 / elem) == 0 ? 16 / elem : 1;
  const int pieces = C / q.vec;
  q.tys = THREADS / (pieces < THREADS ? pieces : THREADS);
  return q;
}

// Rows of a tile, for a launch over n rows: as many blocks as run at once (three times as many where scenes are short, whose
// last tiles are smaller ones), at least four rows a thread.
int tile_rows(int64_t n, int64_t scenes, int tys, int blocks_per_sm) {
  const int64_t side = (int64_t)tys * blocks_per_sm * wcn_num_sms() * (scenes > 16 ? 3 : 1), per = (n + side - 1) / side;
  return (int)((per < 4 ? 4 : per) * tys);
}

size_t sums_smem(int C, int vec) {
  const int pieces = C / vec, txs = pieces < THREADS ? pieces : THREADS, tys = THREADS / txs;
  return ((size_t)2 * tys * txs * vec + 2 * C) * sizeof(float);
}

// The scenes in groups that stay in L2: f(first, behind the last, rows of a tile, tiles).
template <typename F> int in_groups(const int64_t* offsets, int64_t scenes, int64_t row_bytes, bool back, int tys, F&& f) {
  for (int64_t i = 0; i < scenes;) {
    int64_t j = i + 1;
    while (j < scenes && j - i < SCENES && (offsets[j + 1] - offsets[i]) * row_bytes <= GROUP_BYTES) ++j;
    const int rows = tile_rows(offsets[j] - offsets[i], j - i, tys, back ? 1 : 2);
    int64_t tiles = 0;
    for (int64_t k = i; k < j; ++k) tiles += (offsets[k + 1] - offsets[k] + rows - 1) / rows;
    const int rc = tiles ? f(i, j, rows, (int)tiles) : WCN_OK;
    if (rc != WCN_OK) return rc;
    i = j;
  }
  return WCN_OK;
}

template <typename T, int V, int ACT, int SUB> int all_groups(bool back, Params p, const int64_t* offsets, int64_t scenes, cudaStream_t st) {
  const int64_t row_bytes = (int64_t)p.C * sizeof(T) * (back ? 2 : 1);
  const Params base = p;
  const size_t sums = sums_smem(p.C, V), apply = (size_t)2 * p.G * sizeof(float);
  const int pieces = p.C / V, tys = THREADS / (pieces < THREADS ? pieces : THREADS);
  if (sums > 48 * 1024) {
    auto a = group_stats_kernel<T, V>;
    auto b = group_grad_sums_kernel<T, V, ACT, SUB>;
    if (cudaFuncSetAttribute(a, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sums) != cudaSuccess ||
        cudaFuncSetAttribute(b, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sums) != cudaSuccess)
      return WCN_ERR_INITIALIZATION;
  }
  return in_groups(offsets, scenes, row_bytes, back, tys, [&](int64_t i, int64_t j, int rows, int tiles) {
    const int64_t r = offsets[i];
    Scenes s;
    s.count = (int)(j - i);
    int at = 0;
    for (int64_t k = i; k <= j; ++k) {
      s.row0[k - i] = (int)(offsets[k] - r);
      s.tile0[k - i] = at;
      if (k < j) at += (int)((offsets[k + 1] - offsets[k] + rows - 1) / rows);
    }
    p.rows = rows;
    p.x = reinterpret_cast<const T*>(base.x) + r * p.x_ld;
    if (back) p.dy = reinterpret_cast<const T*>(base.dy) + r * p.dy_ld;
    p.out = base.out ? reinterpret_cast<T*>(base.out) + r * p.C : nullptr;
    p.mean = base.mean ? base.mean + i * p.G : nullptr;
    p.rstd = base.rstd ? base.rstd + i * p.G : nullptr;
    if (!back) {
      group_stats_kernel<T, V><<<tiles, THREADS, sums, st>>>(s, p);
      group_apply_kernel<T, V, ACT, SUB><<<tiles, THREADS, apply, st>>>(s, p);
    } else {
      group_grad_sums_kernel<T, V, ACT, SUB><<<tiles, THREADS, sums, st>>>(s, p);
      if (p.out) group_grad_apply_kernel<T, V, ACT, SUB><<<tiles, THREADS, apply, st>>>(s, p);
      if (p.channels) p.channels += (int64_t)tiles * 2 * p.C;   // (the groups' sums are done with, these are not)
    }
    return cudaGetLastError() == cudaSuccess ? WCN_OK : WCN_ERR_EXECUTION;
  });
}

template <typename T, int V, int SUB> int by_act(int act, bool back, const Params& p, const int64_t* offsets, int64_t scenes, cudaStream_t st) {
  switch (act) {
    case NONE: return all_groups<T, V, NONE, SUB>(back, p, offsets, scenes, st);
    case RELU: return all_groups<T, V, RELU, SUB>(back, p, offsets, scenes, st);
    case SILU: return all_groups<T, V, SILU, SUB>(back, p, offsets, scenes, st);
    default: return all_groups<T, V, GELU, SUB>(back, p, offsets, scenes, st);
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

// Tiles of all launches together, and of the largest one.
void count_tiles(const int64_t* offsets, int64_t scenes, int64_t row_bytes, bool back, int tys, int64_t* all, int64_t* most) {
  *all = *most = 0;
  in_groups(offsets, scenes, row_bytes, back, tys, [&](int64_t, int64_t, int, int tiles) {
    *all += tiles;
    if (tiles > *most) *most = tiles;
    return (int)WCN_OK;
  });
}

bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool rows_on16(const void* p, int64_t ld, int elem) { return on16(p) && ld * elem % 16 == 0; }

float from_bits(uint32_t b) {
  float f;
  memcpy(&f, &b, sizeof f);
  return f;
}

// Bytes of the groups' sums (of a launch), then of the channels' (of all of them).
int64_t part_bytes(const int64_t* offsets, int64_t scenes, int C, int G, int elem, bool back, bool channels, int tys, int64_t* total) {
  int64_t all, most;
  count_tiles(offsets, scenes, (int64_t)C * elem * (back ? 2 : 1), back, tys, &all, &most);
  const int64_t first = (most * G * (int64_t)sizeof(float2) + 15) / 16 * 16;
  *total = first + (channels ? all * 2 * C * 4 : 0);
  return first;
}

}  // namespace

extern "C" int wcn_group_norm_workspace_bytes(const int64_t* offsets, int64_t scenes, int32_t channels, int32_t groups, int dtype,
                                              int backward, int64_t* bytes) {
  if (!bytes || !norm_ok(scenes, offsets, channels, groups, dtype)) return WCN_ERR_INVALID_PARAMETERS;
  int64_t most = 0;
  for (int v = 0; v < 2; ++v) {   // (whatever the rows' alignment will be)
    int64_t need;
    const int elem = wcn_dtype_size(dtype);
    part_bytes(offsets, scenes, channels, groups, elem, backward, backward, plan(channels, elem, v).tys, &need);
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
  const Plan q = plan(channels, elem, rows_on16(x, x_ld, elem) && rows_on16(y, channels, elem));
  int64_t need;
  part_bytes(offsets, scenes, channels, groups, elem, false, false, q.tys, &need);
  if (need > workspace_bytes) return WCN_ERR_SCRATCH_TOO_SMALL;
  Params p = {};
  p.x = x; p.out = y; p.gamma = gamma; p.beta = beta; p.mean = mean; p.rstd = rstd; p.part = (float2*)workspace;
  p.x_ld = x_ld; p.C = channels; p.G = groups; p.per = channels / groups; p.eps = from_bits(eps_bits);
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
  const Plan q = plan(channels, elem, rows_on16(x, x_ld, elem) && rows_on16(dy, dy_ld, elem) && rows_on16(dx, channels, elem));
  int64_t need;
  const int64_t first = part_bytes(offsets, scenes, channels, groups, elem, true, sums, q.tys, &need);
  if (need > workspace_bytes) return WCN_ERR_SCRATCH_TOO_SMALL;
  Params p = {};
  p.x = x; p.dy = dy; p.out = dx; p.gamma = gamma; p.beta = beta; p.mean = const_cast<float*>(mean); p.rstd = const_cast<float*>(rstd);
  p.part = (float2*)workspace;
  p.channels = sums ? (float*)((char*)workspace + first) : nullptr;
  p.x_ld = x_ld; p.dy_ld = dy_ld; p.C = channels; p.G = groups; p.per = channels / groups;
  const int rc = by_dtype(dtype, q.vec, act, true, p, offsets, scenes, st);
  if (rc != WCN_OK || !sums) return rc;
  group_param_grads_kernel<<<(2 * channels + 31) / 32, 1024, 0, st>>>(p.channels, (need - first) / (2 * channels * 4), 2 * channels, sums);
  return cudaGetLastError() == cudaSuccess ? WCN_OK : WCN_ERR_EXECUTION;
}
