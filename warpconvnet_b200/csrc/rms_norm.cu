// Root-mean-square norm of [n, channels] rows, with the residual's addition before it:
//     h = round(x + residual),  s = 1 / sqrt(mean_c h^2 + eps),  y = h s w
// its gradients, with u = dy w and xh = h s:
//     dx = dresidual = s (u - xh mean_c(u xh)) + dh,  dw = sum over the rows of dy xh
// and its result in 8 bits: e4m3 codes of y / t with the scale t = max(largest |y| of the row / 448, 2^-126).
//
// Bound by HBM: every row is read once and stays in registers.  L threads share a row (2 to 32 of a warp, or a block of up to
// 1024), V pieces of up to 16 bytes each: the row's sums are a few shuffles.  The norm is that of h as it is written (rounded to the
// rows' type), so that the gradient, which reads it again, is that of the same numbers.  Sums, 1 / sqrt and products are fp32.
// A row whose squares pass the end of fp32 is summed again with its numbers times 2^-66.
// The gradient of w is summed per thread over the rows of a persistent block (tens of them in fp32), then over the block's threads, and
// over the blocks in double by a second launch: no atomics, the same bits on every run.
#include <cuda_fp8.h>

#include "wcn_common.cuh"

namespace {

constexpr int THREADS = 256, MAX_C = 8192, MAX_WARP_C = 1024;
constexpr float LEAST_EPS = 1e-30f;            // beside which squares below the end of fp32 are nothing
constexpr float MOST = 448.f;                  // the largest e4m3 number
constexpr float SMALL = 1.3552527156068805e-20f;   // 2^-66

struct NormParams {
  const void* x;
  const void* residual;   // null: none
  const float* weight;    // null: ones
  void* h;                // with a residual
  void* y;                // null: q and scale are wanted
  uint8_t* q;
  float* scale;
  float* rstd;            // null: not wanted
  int64_t x_ld, res_ld, n;
  int c, lanes;           // threads of a row
  float eps;
  bool plain;             // no norm: codes of x
};

struct GradParams {
  const void* h;
  const void* dy;
  const void* dh;         // null: none
  const float* weight;
  const float* rstd;
  void* dx;               // null: not wanted
  float* partial;         // [blocks][c]; null: no gradient of the weight
  int64_t h_ld, dy_ld, dh_ld, n;
  int c, lanes;
};

// Threads of a block that share a row, at most: 8192 single elements in eights, or 2048 pieces in fours.
constexpr int most_lanes(int e) { return e == 1 ? 1024 : 512; }

// E elements: 16, 8, 4 or 2 bytes.
template <typename T, int E> struct alignas(E * sizeof(T) <= 16 ? E * sizeof(T) : 16) Piece { T v[E]; };
template <typename T, int E> __device__ __forceinline__ Piece<T, E> load_piece(const void* row, int at) {
  return reinterpret_cast<const Piece<T, E>*>(row)[at];
}

// The sum of `v` over the threads of a row.  BLOCK: those of the block.
template <bool BLOCK> __device__ __forceinline__ float row_sum(float v, int lanes, float* part) {
  for (int d = (BLOCK ? 32 : lanes) / 2; d; d >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
  if (!BLOCK) return v;
  const int warps = blockDim.x >> 5;
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.f;
  for (int w = 0; w < warps; ++w) v += part[w];
  return v;
}
template <bool BLOCK> __device__ __forceinline__ uint32_t row_max(uint32_t v, int lanes, uint32_t* part) {
  for (int d = (BLOCK ? 32 : lanes) / 2; d; d >>= 1) v = max(v, __shfl_xor_sync(0xFFFFFFFFu, v, d));
  if (!BLOCK) return v;
  const int warps = blockDim.x >> 5;
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
  for (int w = 0; w < warps; ++w) v = max(v, part[w]);
  return v;
}

template <int E> __device__ __forceinline__ void load_weight(const float* weight, int piece, float (&w)[E]) {
  if (!weight) {
#pragma unroll
    for (int i = 0; i < E; ++i) w[i] = 1.f;
  } else if constexpr (E % 4 == 0) {
#pragma unroll
    for (int i = 0; i < E; i += 4) *reinterpret_cast<float4*>(w + i) = __ldg(reinterpret_cast<const float4*>(weight + piece * E + i));
  } else {
    w[0] = __ldg(weight + piece);
  }
}

template <typename T, int E, int V, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? most_lanes(E) : THREADS) rms_norm_kernel(const __grid_constant__ NormParams p) {
  __shared__ uint32_t part[32];
  const int lanes = BLOCK ? (int)blockDim.x : p.lanes, lane = threadIdx.x % lanes, rows = (int)blockDim.x / lanes, pieces = p.c / E;
  const int64_t row = (int64_t)blockIdx.x * rows + threadIdx.x / lanes;
  const bool live = row < p.n;      // (threads of no row take part in the shuffles)
  Piece<T, E> h[V];
  const T* const x = reinterpret_cast<const T*>(p.x) + (live ? row : 0) * p.x_ld;
  const T* const r = p.residual ? reinterpret_cast<const T*>(p.residual) + (live ? row : 0) * p.res_ld : nullptr;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int at = lane + j * lanes;
    if (live && at < pieces) {
      h[j] = load_piece<T, E>(x, at);
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) h[j].v[i] = wcn_from_float<T>(0.f);
    }
  }
  if (r) {
    Piece<T, E> more[V];
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (live && lane + j * lanes < pieces) more[j] = load_piece<T, E>(r, lane + j * lanes);
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (live && lane + j * lanes < pieces) {
#pragma unroll
        for (int i = 0; i < E; ++i) h[j].v[i] = wcn_from_float<T>(wcn_to_float<T>(h[j].v[i]) + wcn_to_float<T>(more[j].v[i]));
        reinterpret_cast<Piece<T, E>*>(reinterpret_cast<T*>(p.h) + row * p.c)[lane + j * lanes] = h[j];
      }
  }
  float s = 1.f;
  if (!p.plain) {
    auto squares = [&](float by) {
      float t[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < V; ++j)
#pragma unroll
        for (int i = 0; i < E; ++i) {
          const float v = wcn_to_float<T>(h[j].v[i]) * by;
          t[i & 3] = fmaf(v, v, t[i & 3]);
        }
      return row_sum<BLOCK>((t[0] + t[1]) + (t[2] + t[3]), lanes, reinterpret_cast<float*>(part));
    };
    const float sum = squares(1.f);
    s = 1.f / sqrtf(sum / (float)p.c + p.eps);
    const bool over = sum == INFINITY;
    if (BLOCK ? over : __any_sync(0xFFFFFFFFu, over)) {   // (one answer for all threads that sum together)
      const float again = squares(SMALL);
      if (over) s = SMALL / sqrtf(again / (float)p.c);
    }
    if (p.rstd && live && lane == 0) p.rstd[row] = s;
  }
  if (p.y) {
    if (!live) return;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int at = lane + j * lanes;
      if (at >= pieces) continue;
      float w[E];
      load_weight<E>(p.weight, at, w);
      Piece<T, E> y;
#pragma unroll
      for (int i = 0; i < E; ++i) y.v[i] = wcn_from_float<T>(wcn_to_float<T>(h[j].v[i]) * s * w[i]);
      reinterpret_cast<Piece<T, E>*>(reinterpret_cast<T*>(p.y) + row * p.c)[at] = y;
    }
    return;
  }
  float y[V][E];
  uint32_t most = 0;      // of |y| as bits: what is no number lies above all numbers
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int at = lane + j * lanes;
    float w[E];
    if (at < pieces) load_weight<E>(p.weight, at, w);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      y[j][i] = at < pieces ? wcn_to_float<T>(h[j].v[i]) * s * w[i] : 0.f;
      most = max(most, __float_as_uint(y[j][i]) & 0x7FFFFFFFu);
    }
  }
  most = row_max<BLOCK>(most, lanes, part);
  if (!live) return;
  const float scale = most >= 0x7F800000u ? __int_as_float(0x7FC00000) : fmaxf(__uint_as_float(most) * (1.f / MOST), 1.17549435e-38f);
  const float inverse = 1.f / scale;
  if (lane == 0) p.scale[row] = scale;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int at = lane + j * lanes;
    if (at >= pieces) continue;
    Piece<uint8_t, E> q;
#pragma unroll
    for (int i = 0; i < E; ++i) q.v[i] = __nv_cvt_float_to_fp8(y[j][i] * inverse, __NV_SATFINITE, __NV_E4M3);
    reinterpret_cast<Piece<uint8_t, E>*>(p.q + row * p.c)[at] = q;
  }
}

template <typename T, int E, int V, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? most_lanes(E) : THREADS) rms_norm_backward_kernel(const __grid_constant__ GradParams p) {
  __shared__ float part[32];
  __shared__ float sums[BLOCK ? 1 : (THREADS / 32) * MAX_WARP_C];
  const int lanes = BLOCK ? (int)blockDim.x : p.lanes, lane = threadIdx.x % lanes, rows = (int)blockDim.x / lanes, pieces = p.c / E;
  float dw[V][E];
#pragma unroll
  for (int j = 0; j < V; ++j)
#pragma unroll
    for (int i = 0; i < E; ++i) dw[j][i] = 0.f;
  const float over_c = 1.f / (float)p.c;
  for (int64_t first = (int64_t)blockIdx.x * rows; first < p.n; first += (int64_t)gridDim.x * rows) {
    const int64_t row = first + threadIdx.x / lanes;
    const bool live = row < p.n;
    const int64_t from = live ? row : 0;
    Piece<T, E> h[V], dy[V], dh[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int at = lane + j * lanes;
      if (!live || at >= pieces) continue;
      h[j] = load_piece<T, E>(reinterpret_cast<const T*>(p.h) + from * p.h_ld, at);
      dy[j] = load_piece<T, E>(reinterpret_cast<const T*>(p.dy) + from * p.dy_ld, at);
      if (p.dh) dh[j] = load_piece<T, E>(reinterpret_cast<const T*>(p.dh) + from * p.dh_ld, at);
    }
    const float s = live ? __ldg(&p.rstd[row]) : 0.f;
    float t = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int at = lane + j * lanes;
      if (!live || at >= pieces) continue;
      float w[E];
      load_weight<E>(p.weight, at, w);
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const float xh = wcn_to_float<T>(h[j].v[i]) * s, g = wcn_to_float<T>(dy[j].v[i]);
        t = fmaf(g * w[i], xh, t);
        dw[j][i] = fmaf(g, xh, dw[j][i]);
      }
    }
    t = row_sum<BLOCK>(t, lanes, part) * over_c;
    if (!p.dx || !live) continue;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int at = lane + j * lanes;
      if (at >= pieces) continue;
      float w[E];
      load_weight<E>(p.weight, at, w);
      Piece<T, E> dx;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const float xh = wcn_to_float<T>(h[j].v[i]) * s;
        float v = s * fmaf(-xh, t, wcn_to_float<T>(dy[j].v[i]) * w[i]);
        if (p.dh) v += wcn_to_float<T>(dh[j].v[i]);
        dx.v[i] = wcn_from_float<T>(v);
      }
      reinterpret_cast<Piece<T, E>*>(reinterpret_cast<T*>(p.dx) + row * p.c)[at] = dx;
    }
  }
  if (!p.partial) return;
  float* const out = p.partial + (int64_t)blockIdx.x * p.c;
  if (BLOCK) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int at = lane + j * lanes;
      if (at >= pieces) continue;
#pragma unroll
      for (int i = 0; i < E; ++i) out[at * E + i] = dw[j][i];
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int at = lane + j * lanes;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      float v = dw[j][i];
      for (int d = lanes; d < 32; d <<= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
      if ((threadIdx.x & 31) < lanes && at < pieces) sums[(threadIdx.x >> 5) * MAX_WARP_C + at * E + i] = v;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < p.c; i += THREADS) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) v += sums[w * MAX_WARP_C + i];
    out[i] = v;
  }
}

// dw from the blocks' sums: 32 channels a block, eight threads that share the blocks.
__global__ void __launch_bounds__(256) rms_norm_weight_kernel(const float* __restrict__ partial, int blocks, int c, float* __restrict__ out) {
  __shared__ double part[8][32];
  const int i = blockIdx.x * 32 + (threadIdx.x & 31), side = threadIdx.x >> 5;
  double v = 0;
  if (i < c)
#pragma unroll 8
    for (int b = side; b < blocks; b += 8) v += (double)__ldg(&partial[(int64_t)b * c + i]);
  part[side][threadIdx.x & 31] = v;
  __syncthreads();
  if (side || i >= c) return;
  for (int s = 1; s < 8; ++s) v += part[s][threadIdx.x];
  out[i] = (float)v;
}

// How a row is divided: E elements a piece (as far as the rows' starts allow), V pieces a thread, `lanes` threads.
struct Plan {
  int e, v, lanes;
  bool block;
};
Plan plan_row(int c, int e) {
  const int pieces = c / e;
  Plan best = {e, 0, 0, false};
  if (pieces <= 32 * 4) {   // threads of one warp: the least idle pieces; several a thread, so that loads are in flight
    int least = INT_MAX;
    for (int lanes = 32; lanes >= 1; lanes /= 2) {
      const int v = (pieces + lanes - 1) / lanes;
      if (v > 4 || (lanes == 1 && pieces > 1)) break;
      const int cost = lanes * v * 4 - (v < 3 ? v : 3);
      if (cost < least) { least = cost; best.v = v; best.lanes = lanes; }
    }
    return best;
  }
  best.block = true;
  best.lanes = 64;
  while (best.lanes < most_lanes(e) && best.lanes * 4 < pieces) best.lanes *= 2;
  best.v = (pieces + best.lanes - 1) / best.lanes <= 4 ? 4 : 8;
  return best;
}

bool row_fits(const void* p, int64_t ld, int64_t n, int e, int size) {
  return !p || (reinterpret_cast<uintptr_t>(p) % (e * size) == 0 && (n <= 1 || ld % e == 0));
}

#define WCN_ROW_CASES(RUN)                                                                 \
  if (plan.block) {                                                                        \
    if (plan.v == 8) { if constexpr (E == 1) RUN(8, true); } else RUN(4, true);            \
  } else {                                                                                 \
    switch (plan.v) {                                                                      \
      case 1: RUN(1, false); break;                                                        \
      case 2: RUN(2, false); break;                                                        \
      case 3: RUN(3, false); break;                                                        \
      default: RUN(4, false); break;                                                       \
    }                                                                                      \
  }

template <typename T, int E> int norm_with(const NormParams& q, cudaStream_t st) {
  const Plan plan = plan_row(q.c, E);
  NormParams p = q;
  p.lanes = plan.lanes;
  const int threads = plan.block ? plan.lanes : THREADS, rows = threads / plan.lanes;
  const unsigned grid = (unsigned)((p.n + rows - 1) / rows);
#define RUN(V, B) rms_norm_kernel<T, E, V, B><<<grid, threads, 0, st>>>(p)
  WCN_ROW_CASES(RUN)
#undef RUN
  WCN_CHECK_LAUNCH();
  return WCN_OK;
}

// Elements of a piece with which all rows start on its boundaries: 16, 8 bytes or one element.
template <typename T> int elements(const NormParams& p) {
  for (int e = 16 / (int)sizeof(T); e >= 4; e /= 2)
    if (p.c % e == 0 && row_fits(p.x, p.x_ld, p.n, e, sizeof(T)) && row_fits(p.residual, p.res_ld, p.n, e, sizeof(T)) && row_fits(p.h, e, 1, e, sizeof(T)) &&
        row_fits(p.y, e, 1, e, sizeof(T)) && row_fits(p.q, e, 1, e, 1) && row_fits(p.weight, 4, 1, 4, 4))
      return e;
  return 1;
}
template <typename T> int elements(const GradParams& p) {
  for (int e = 16 / (int)sizeof(T); e >= 4; e /= 2)
    if (p.c % e == 0 && row_fits(p.h, p.h_ld, p.n, e, sizeof(T)) && row_fits(p.dy, p.dy_ld, p.n, e, sizeof(T)) && row_fits(p.dh, p.dh_ld, p.n, e, sizeof(T)) &&
        row_fits(p.dx, e, 1, e, sizeof(T)) && row_fits(p.weight, 4, 1, 4, 4))
      return e;
  return 1;
}

template <typename T> int norm_as(const NormParams& p, cudaStream_t st) {
  const int e = elements<T>(p);
  if (sizeof(T) == 2 && e == 8) return norm_with<T, sizeof(T) == 2 ? 8 : 4>(p, st);
  return e == 4 ? norm_with<T, 4>(p, st) : norm_with<T, 1>(p, st);
}
int norm(const NormParams& p, int dtype, cudaStream_t st) {
  if (dtype == WCN_F32) return norm_as<float>(p, st);
  return dtype == WCN_F16 ? norm_as<__half>(p, st) : norm_as<__nv_bfloat16>(p, st);
}

// Persistent blocks: four of 256 threads a multiprocessor (registers), two of a row each; at least four rows a thread where sums are wanted.
int grad_blocks(int64_t n, int rows) {
  const int64_t want = (n + 4 * rows - 1) / (4 * (int64_t)rows), most = 4 * (int64_t)wcn_num_sms();
  return (int)(want < 1 ? 1 : want < most ? want : most);
}

template <typename T, int E> int grad_with(const GradParams& q, float* dweight, cudaStream_t st) {
  const Plan plan = plan_row(q.c, E);
  GradParams p = q;
  p.lanes = plan.lanes;
  const int threads = plan.block ? plan.lanes : THREADS, blocks = grad_blocks(p.n, threads / plan.lanes);
#define RUN(V, B) rms_norm_backward_kernel<T, E, V, B><<<blocks, threads, 0, st>>>(p)
  WCN_ROW_CASES(RUN)
#undef RUN
  wcn_launched = 1;
  if (p.partial) {
    rms_norm_weight_kernel<<<(p.c + 31) / 32, 256, 0, st>>>(p.partial, blocks, p.c, dweight);
    ++wcn_launched;
  }
  WCN_CHECK_LAUNCH();
  return WCN_OK;
}
template <typename T> int grad_as(const GradParams& p, float* dweight, cudaStream_t st) {
  const int e = elements<T>(p);
  if (sizeof(T) == 2 && e == 8) return grad_with<T, sizeof(T) == 2 ? 8 : 4>(p, dweight, st);
  return e == 4 ? grad_with<T, 4>(p, dweight, st) : grad_with<T, 1>(p, dweight, st);
}

bool sizes_taken(int64_t n, int c, int dtype) {
  return n >= 0 && n <= 0x7FFFFEFF && c >= 1 && c <= MAX_C && dtype >= WCN_F32 && dtype <= WCN_BF16;
}
float float_of(uint32_t bits) {
  union { uint32_t u; float f; } v = {bits};
  return v.f;
}

}  // namespace

extern "C" int wcn_rms_norm(const void* x, int64_t x_ld, const void* residual, int64_t residual_ld, int64_t n, int32_t channels, int dtype,
                            const float* weight, uint32_t eps_bits, void* h, void* y, float* rstd, void* q, float* scale, void* stream) {
  if (!sizes_taken(n, channels, dtype)) return WCN_ERR_INVALID_PARAMETERS;
  if (n == 0) return WCN_OK;
  if (!(float_of(eps_bits) >= LEAST_EPS)) return WCN_ERR_INVALID_PARAMETERS;
  if (!x || (residual && !h) || !y == !q || (q && !scale) || (n > 1 && (x_ld < channels || (residual && residual_ld < channels)))) return WCN_ERR_INVALID_PARAMETERS;
  NormParams p = {x, residual, weight, residual ? h : nullptr, y, (uint8_t*)q, scale, rstd, x_ld, residual_ld, n, channels, 0, float_of(eps_bits), false};
  return norm(p, dtype, wcn_stream(stream));
}

extern "C" int wcn_quantize_rows(const void* x, int64_t x_ld, int64_t n, int32_t channels, int dtype, void* q, float* scale, void* stream) {
  if (!sizes_taken(n, channels, dtype)) return WCN_ERR_INVALID_PARAMETERS;
  if (n == 0) return WCN_OK;
  if (!x || !q || !scale || (n > 1 && x_ld < channels)) return WCN_ERR_INVALID_PARAMETERS;
  NormParams p = {x, nullptr, nullptr, nullptr, nullptr, (uint8_t*)q, scale, nullptr, x_ld, 0, n, channels, 0, 0.f, true};
  return norm(p, dtype, wcn_stream(stream));
}

extern "C" int wcn_rms_norm_workspace_bytes(int64_t n, int32_t channels, int64_t* bytes) {
  if (!bytes || !sizes_taken(n, channels, WCN_F32)) return WCN_ERR_INVALID_PARAMETERS;
  *bytes = (int64_t)grad_blocks(n, 1) * channels * 4;   // (rows of a block: one at least)
  return WCN_OK;
}

extern "C" int wcn_rms_norm_backward(const void* h, int64_t h_ld, const void* dy, int64_t dy_ld, const void* dh, int64_t dh_ld, int64_t n,
                                     int32_t channels, int dtype, const float* weight, const float* rstd, void* dx, float* dweight,
                                     void* workspace, int64_t workspace_bytes, void* stream) {
  if (!sizes_taken(n, channels, dtype)) return WCN_ERR_INVALID_PARAMETERS;
  int64_t need = 0;
  wcn_rms_norm_workspace_bytes(n, channels, &need);
  if (n == 0 || !h || !dy || !rstd || (!dx && !dweight) || (n > 1 && (h_ld < channels || dy_ld < channels || (dh && dh_ld < channels))))
    return WCN_ERR_INVALID_PARAMETERS;
  if (dweight && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 3) || workspace_bytes < need)) return WCN_ERR_INVALID_PARAMETERS;
  GradParams p = {h, dy, dh, weight, rstd, dx, dweight ? (float*)workspace : nullptr, h_ld, dy_ld, dh_ld, n, channels, 0};
  cudaStream_t st = wcn_stream(stream);
  if (dtype == WCN_F32) return grad_as<float>(p, dweight, st);
  return dtype == WCN_F16 ? grad_as<__half>(p, dweight, st) : grad_as<__nv_bfloat16>(p, dweight, st);
}
