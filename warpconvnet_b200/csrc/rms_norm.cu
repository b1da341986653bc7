// Root-mean-square norm of [n, channels] rows, with the residual's addition before it:
//     h = round(x + residual),  s = 1 / sqrt(mean_c h^2 + eps),  y = h s w
// its gradients, with u = dy w and xh = h s:
//     dx = dresidual = s (u - xh mean_c(u xh)) + dh,  dw = sum over the rows of dy xh
// and its result in 8 bits: e4m3 codes of y / t with the scale t = max(largest |y| of the row / 448, 2^-126).
//
// Bound by HBM: every row is read once and stays in registers.  L threads share a row (2 to 32 of a warp, or a block of up to
// 1024), V pieces of up to 16 bytes each: the row's sums are a few shuffles.  The norm is that of h as it is written (rounded to the
// rows' type), so that the gradient, which reads it again, is that of the same numbers.  Sums, 1 / sqrt and products are fp32.
// A row whose squares pass the end of fp32 is summed again with its numbers times 2^-80: 8192 of the largest, 2^128 each, then have
// squares of 2^109 in all, and those that the first sum could not hold, 2^128, are 2^-32.
// The gradient of w is summed in fp32 per thread over the rows of a persistent block (25 of 240 000 x 96 in 16 bits, 130 of 1 200 000; more
// with more rows), then over the block's threads, and over the blocks in double by a second launch: no atomics, the same bits on every run.
// 240 000 x 96 bf16 with residual 28 us forward (184 MB at 6.6 TB/s, some of what is written still in L2), 46 + 7 backward (161 MB, 4.0
// TB/s: the loads in flight are those of 32 warps, a row and the next one each); 1 200 000 x 96 fp16 into 8 bits 120 (811 MB, 6.8 TB/s).
#include <cuda_fp8.h>

#include <type_traits>

#include "wcn_common.cuh"

namespace {

constexpr int THREADS = 256, MAX_C = 8192, MAX_WARP_C = 512;   // (channels of a warp's row in the gradient)
constexpr float LEAST_EPS = 1e-30f;            // beside which squares below the end of fp32 are nothing
constexpr float MOST = 448.f;                  // the largest e4m3 number
constexpr float SMALL = 8.271806125530277e-25f;   // 2^-80

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

// E elements, 16, 8, 4 or 2 bytes, in registers as they come: an array of 16-bit numbers would be moved one by one (a third of the
// instructions of the gradient).
template <typename T, int E> struct Piece {
  static constexpr int BYTES = E * (int)sizeof(T), WORDS = BYTES > 4 ? BYTES / 4 : 1, PAIRS = (E + 1) / 2;   // (a single number has nothing beside it)
  uint32_t w[WORDS];

  __device__ __forceinline__ void load(const T* row, int at) {
    if constexpr (BYTES == 16) {
      const uint4 v = reinterpret_cast<const uint4*>(row)[at];
      w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else if constexpr (BYTES == 8) {
      const uint2 v = reinterpret_cast<const uint2*>(row)[at];
      w[0] = v.x; w[1] = v.y;
    } else if constexpr (BYTES == 4) {
      w[0] = reinterpret_cast<const uint32_t*>(row)[at];
    } else {
      w[0] = reinterpret_cast<const uint16_t*>(row)[at];
    }
  }
  __device__ __forceinline__ void store(T* row, int at) const {
    if constexpr (BYTES == 16) reinterpret_cast<uint4*>(row)[at] = make_uint4(w[0], w[1], w[2], w[3]);
    else if constexpr (BYTES == 8) reinterpret_cast<uint2*>(row)[at] = make_uint2(w[0], w[1]);
    else if constexpr (BYTES == 4) reinterpret_cast<uint32_t*>(row)[at] = w[0];
    else reinterpret_cast<uint16_t*>(row)[at] = (uint16_t)w[0];
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) w[i] = 0u;
  }
  // Numbers 2 i and 2 i + 1.
  __device__ __forceinline__ float2 pair(int i) const {
    if constexpr (sizeof(T) == 4) return make_float2(__uint_as_float(w[2 * i]), E > 1 ? __uint_as_float(w[2 * i + (E > 1)]) : 0.f);
    else if constexpr (std::is_same<T, __nv_bfloat16>::value) return make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
    else return __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
  }
  __device__ __forceinline__ void set(int i, float2 v) {
    if constexpr (sizeof(T) == 4) {
      w[2 * i] = __float_as_uint(v.x);
      if constexpr (E > 1) w[2 * i + 1] = __float_as_uint(v.y);
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      const __nv_bfloat162 t = __float22bfloat162_rn(v);
      w[i] = *reinterpret_cast<const uint32_t*>(&t);
    } else {
      const __half2 t = __float22half2_rn(v);
      w[i] = *reinterpret_cast<const uint32_t*>(&t);
    }
  }
};
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

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

template <int E> __device__ __forceinline__ void load_weight(const float* weight, int piece, float2 (&w)[(E + 1) / 2]) {
  if (!weight) {
#pragma unroll
    for (int i = 0; i < (E + 1) / 2; ++i) w[i] = both(1.f);
  } else if constexpr (E % 4 == 0) {
#pragma unroll
    for (int i = 0; i < E / 4; ++i) {
      const float4 t = __ldg(reinterpret_cast<const float4*>(weight + piece * E) + i);
      w[2 * i] = make_float2(t.x, t.y);
      w[2 * i + 1] = make_float2(t.z, t.w);
    }
  } else {
    w[0] = make_float2(__ldg(weight + piece), 0.f);
  }
}

template <typename T, int E, int V, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? most_lanes(E) : THREADS) rms_norm_kernel(const __grid_constant__ NormParams p) {
  __shared__ uint32_t part[32];
  constexpr int P = Piece<T, E>::PAIRS;
  const int lanes = BLOCK ? (int)blockDim.x : p.lanes, lane = threadIdx.x % lanes, rows = (int)blockDim.x / lanes, pieces = p.c / E;
  const int64_t row = (int64_t)blockIdx.x * rows + threadIdx.x / lanes;
  const bool live = row < p.n;      // (threads of no row take part in the shuffles)
  Piece<T, E> h[V];
  const T* const x = reinterpret_cast<const T*>(p.x) + (live ? row : 0) * p.x_ld;
  const T* const r = p.residual ? reinterpret_cast<const T*>(p.residual) + (live ? row : 0) * p.res_ld : nullptr;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int at = lane + j * lanes;
    if (live && at < pieces) h[j].load(x, at);
    else h[j].zero();
  }
  if (r) {
    Piece<T, E> more[V];
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (live && lane + j * lanes < pieces) more[j].load(r, lane + j * lanes);
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (live && lane + j * lanes < pieces) {
#pragma unroll
        for (int i = 0; i < P; ++i) h[j].set(i, __fadd2_rn(h[j].pair(i), more[j].pair(i)));
        h[j].store(reinterpret_cast<T*>(p.h) + row * p.c, lane + j * lanes);
      }
  }
  float s = 1.f;
  if (!p.plain) {
    auto squares = [&](float by) {
      float2 t[2] = {both(0.f), both(0.f)};
#pragma unroll
      for (int j = 0; j < V; ++j)
#pragma unroll
        for (int i = 0; i < P; ++i) {
          const float2 v = __fmul2_rn(h[j].pair(i), both(by));
          t[i & 1] = __ffma2_rn(v, v, t[i & 1]);
        }
      return row_sum<BLOCK>((t[0].x + t[0].y) + (t[1].x + t[1].y), lanes, reinterpret_cast<float*>(part));
    };
    const float mean = squares(1.f) / (float)p.c + p.eps;
    s = 1.f / sqrtf(mean);
    const bool over = mean == INFINITY;
    if (BLOCK ? over : __any_sync(0xFFFFFFFFu, over)) {   // (one answer for all threads that sum together)
      const float again = squares(SMALL);
      if (over) s = SMALL / sqrtf(again / (float)p.c + p.eps * SMALL * SMALL);
    }
    if (p.rstd && live && lane == 0) p.rstd[row] = s;
  }
  if (p.y) {
    if (!live) return;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int at = lane + j * lanes;
      if (at >= pieces) continue;
      float2 w[P];
      load_weight<E>(p.weight, at, w);
      Piece<T, E> y;
#pragma unroll
      for (int i = 0; i < P; ++i) y.set(i, __fmul2_rn(__fmul2_rn(h[j].pair(i), both(s)), w[i]));
      y.store(reinterpret_cast<T*>(p.y) + row * p.c, at);
    }
    return;
  }
  float2 y[V][P];
  uint32_t most = 0;      // of |y| as bits: what is no number lies above all numbers
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int at = lane + j * lanes;
    float2 w[P];
    if (at < pieces) load_weight<E>(p.weight, at, w);
#pragma unroll
    for (int i = 0; i < P; ++i) {
      y[j][i] = at < pieces ? __fmul2_rn(__fmul2_rn(h[j].pair(i), both(s)), w[i]) : both(0.f);
      most = max(most, __float_as_uint(y[j][i].x) & 0x7FFFFFFFu);
      if (E > 1) most = max(most, __float_as_uint(y[j][i].y) & 0x7FFFFFFFu);
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
    uint8_t* const q = p.q + row * p.c;
    if constexpr (E == 1) {
      q[at] = __nv_cvt_float_to_fp8(y[j][0].x * inverse, __NV_SATFINITE, __NV_E4M3);
    } else {
      uint32_t words[E / 4];
#pragma unroll
      for (int i = 0; i < E / 4; ++i) {
        const uint32_t low = __nv_cvt_float2_to_fp8x2(__fmul2_rn(y[j][2 * i], both(inverse)), __NV_SATFINITE, __NV_E4M3);
        const uint32_t high = __nv_cvt_float2_to_fp8x2(__fmul2_rn(y[j][2 * i + 1], both(inverse)), __NV_SATFINITE, __NV_E4M3);
        words[i] = low | high << 16;
      }
      if constexpr (E == 8) reinterpret_cast<uint2*>(q)[at] = make_uint2(words[0], words[1]);
      else reinterpret_cast<uint32_t*>(q)[at] = words[0];
    }
  }
}

// Rows of up to 64 pieces are a part of a warp's, one piece a thread or two: the weights and the sums for their gradient stay in
// registers, 64 of them with one piece, so that 32 warps are resident.  (Three pieces of four threads, 96 channels in 16 bits, took 56 us
// for 240 000 rows.)
constexpr int resident_blocks(int v) { return v == 1 ? 4 : 2; }
template <typename T, int E, int V, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? most_lanes(E) : THREADS, BLOCK ? 1 : resident_blocks(V)) rms_norm_backward_kernel(const __grid_constant__ GradParams p) {
  __shared__ float part[32];
  __shared__ float sums[BLOCK ? 1 : (THREADS / 32) * MAX_WARP_C];
  const int lanes = BLOCK ? (int)blockDim.x : p.lanes, lane = threadIdx.x % lanes, rows = (int)blockDim.x / lanes, pieces = p.c / E;
  constexpr bool AHEAD = V <= 2;   // the next row's pieces are on their way while this one's are used, as far as registers go
  constexpr int P = Piece<T, E>::PAIRS;
  float2 dw[V][P], w[V][P];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    if (lane + j * lanes < pieces) load_weight<E>(p.weight, lane + j * lanes, w[j]);
#pragma unroll
    for (int i = 0; i < P; ++i) dw[j][i] = both(0.f);
  }
  const float over_c = 1.f / (float)p.c;
  Piece<T, E> h[V], dy[V], dh[V], next_h[V], next_dy[V], next_dh[V];
  float s = 0.f, next_s = 0.f;
  const int64_t step = (int64_t)gridDim.x * rows;
  auto request = [&](int64_t row) {
    if (row >= p.n) return;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int at = lane + j * lanes;
      if (at >= pieces) continue;
      next_h[j].load(reinterpret_cast<const T*>(p.h) + row * p.h_ld, at);
      next_dy[j].load(reinterpret_cast<const T*>(p.dy) + row * p.dy_ld, at);
      if (p.dh) next_dh[j].load(reinterpret_cast<const T*>(p.dh) + row * p.dh_ld, at);
    }
    next_s = __ldg(&p.rstd[row]);
  };
  if (AHEAD) request((int64_t)blockIdx.x * rows + threadIdx.x / lanes);
  for (int64_t first = (int64_t)blockIdx.x * rows; first < p.n; first += step) {
    const int64_t row = first + threadIdx.x / lanes;
    const bool live = row < p.n;
    if (!AHEAD) request(row);
#pragma unroll
    for (int j = 0; j < V; ++j) { h[j] = next_h[j]; dy[j] = next_dy[j]; dh[j] = next_dh[j]; }
    s = next_s;
    if (AHEAD) request(row + step);
    float2 sum = both(0.f);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (!live || lane + j * lanes >= pieces) continue;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const float2 xh = __fmul2_rn(h[j].pair(i), both(s)), g = dy[j].pair(i);
        sum = __ffma2_rn(__fmul2_rn(g, w[j][i]), xh, sum);
        dw[j][i] = __ffma2_rn(g, xh, dw[j][i]);
      }
    }
    const float t = row_sum<BLOCK>(E > 1 ? sum.x + sum.y : sum.x, lanes, part) * over_c;
    if (!p.dx || !live) continue;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int at = lane + j * lanes;
      if (at >= pieces) continue;
      Piece<T, E> dx;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const float2 xh = __fmul2_rn(h[j].pair(i), both(s)), d = __ffma2_rn(xh, both(-t), __fmul2_rn(dy[j].pair(i), w[j][i]));
        dx.set(i, p.dh ? __ffma2_rn(d, both(s), dh[j].pair(i)) : __fmul2_rn(d, both(s)));
      }
      dx.store(reinterpret_cast<T*>(p.dx) + row * p.c, at);
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
      for (int i = 0; i < E; ++i) out[at * E + i] = i & 1 ? dw[j][i / 2].y : dw[j][i / 2].x;
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int at = lane + j * lanes;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      float v = i & 1 ? dw[j][i / 2].y : dw[j][i / 2].x;
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

// dw from the blocks' sums: 32 channels a block, 32 threads that share the blocks (eight took 14 us for 592 blocks and 96 channels).
constexpr int SIDES = 32;
__global__ void __launch_bounds__(32 * SIDES) rms_norm_weight_kernel(const float* __restrict__ partial, int blocks, int c, float* __restrict__ out) {
  __shared__ double part[SIDES][32];
  const int i = blockIdx.x * 32 + (threadIdx.x & 31), side = threadIdx.x >> 5;
  double v = 0;
  if (i < c)
#pragma unroll 8
    for (int b = side; b < blocks; b += SIDES) v += (double)__ldg(&partial[(int64_t)b * c + i]);
  part[side][threadIdx.x & 31] = v;
  __syncthreads();
  if (side || i >= c) return;
  for (int s = 1; s < SIDES; ++s) v += part[s][threadIdx.x];
  out[i] = (float)v;
}

// How a row is divided: E elements a piece (as far as the rows' starts allow), V pieces a thread, `lanes` threads.
struct Plan {
  int e, v, lanes;
  bool block;
};
// `most`: pieces of a thread of a warp's row at most.
Plan plan_row(int c, int e, int most) {
  const int pieces = c / e;
  Plan best = {e, 0, 0, false};
  if (most == 2 && pieces <= 64) {   // (the gradient: registers)
    best.lanes = 1;
    while (best.lanes < 32 && best.lanes < pieces) best.lanes *= 2;
    best.v = pieces <= 32 ? 1 : 2;
    return best;
  }
  if (pieces <= 32 * most) {   // threads of one warp: the least idle pieces; several a thread, so that loads are in flight
    int least = INT_MAX;
    for (int lanes = 32; lanes >= 1; lanes /= 2) {
      const int v = (pieces + lanes - 1) / lanes;
      if (v > most || (lanes == 1 && pieces > 1)) break;
      const int cost = lanes * v * 4 - (v < 3 ? v : 3);
      if (cost < least) { least = cost; best.v = v; best.lanes = lanes; }
    }
    return best;
  }
  best.block = true;
  best.lanes = 64;
  const int each = most == 2 && pieces <= 1024 ? 2 : 4;
  while (best.lanes < most_lanes(e) && best.lanes * each < pieces) best.lanes *= 2;
  best.v = (pieces + best.lanes - 1) / best.lanes <= each ? each : 8;
  return best;
}

bool row_fits(const void* p, int64_t ld, int64_t n, int e, int size) {
  return !p || (reinterpret_cast<uintptr_t>(p) % (e * size) == 0 && (n <= 1 || ld % e == 0));
}

#define WCN_ROW_CASES(RUN)                                                                 \
  if (plan.block) {                                                                        \
    if (plan.v == 8) { if constexpr (E == 1) RUN(8, true); } else if (plan.v == 4) RUN(4, true); else RUN(2, true); \
  } else {                                                                                 \
    switch (plan.v) {                                                                      \
      case 1: RUN(1, false); break;                                                        \
      case 2: RUN(2, false); break;                                                        \
      case 3: if constexpr (MOST > 2) RUN(3, false); break;                                \
      default: if constexpr (MOST > 2) RUN(4, false); break;                               \
    }                                                                                      \
  }

template <typename T, int E> int norm_with(const NormParams& q, cudaStream_t st) {
  constexpr int MOST = 4;
  const Plan plan = plan_row(q.c, E, MOST);
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

// Persistent blocks, as many as are resident: 1024 threads a multiprocessor, with more than a piece 512 (registers).  At least four rows a
// thread, so that few sums are left.
int grad_blocks(int64_t n, int rows, int threads, int v) {
  const int64_t want = (n + 4 * rows - 1) / (4 * (int64_t)rows), room = v == 1 ? 1024 : 512;
  const int64_t most = (room > threads ? room / threads : 1) * wcn_num_sms();
  return (int)(want < 1 ? 1 : want < most ? want : most);
}

template <typename T, int E> int grad_with(const GradParams& q, float* dweight, cudaStream_t st) {
  constexpr int MOST = 2;
  const Plan plan = plan_row(q.c, E, MOST);
  GradParams p = q;
  p.lanes = plan.lanes;
  const int threads = plan.block ? plan.lanes : THREADS, blocks = grad_blocks(p.n, threads / plan.lanes, threads, plan.v);
#define RUN(V, B) rms_norm_backward_kernel<T, E, V, B><<<blocks, threads, 0, st>>>(p)
  WCN_ROW_CASES(RUN)
#undef RUN
  wcn_launched = 1;
  if (p.partial) {
    rms_norm_weight_kernel<<<(p.c + 31) / 32, 32 * SIDES, 0, st>>>(p.partial, blocks, p.c, dweight);
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
  if (!(float_of(eps_bits) >= LEAST_EPS) || float_of(eps_bits) == INFINITY) return WCN_ERR_INVALID_PARAMETERS;
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
  *bytes = (int64_t)grad_blocks(n, 1, 64, 1) * channels * 4;   // (rows and threads of a block: as few as they may be)
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
