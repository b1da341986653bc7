// Tiles of fp32 products on the FMA pipes, shared by the kernels of linear layers.  Everything is in an unnamed namespace: each
// translation unit gets its own copy.
#pragma once
#include "wcn_common.cuh"

namespace {

constexpr int FP32_THREADS = 256;
constexpr int TILE = 64, DEPTH = 16, CHAIN = 128;   // a chain of 128 products has a sum of its own

enum Layout { LOGITS = 0, ROWS_BY_CLASSES = 1, CLASSES_BY_ROWS = 2 };   // A[m][k] B[n][k]; A[m][k] B[k][n]; A[k][m] B[k][n]

// One tile of 64 x 64 sums over k in [k0, k1): a thread has rows ty * 4 .. and columns tx * 4 ..; `sums`: A's row sums (tx = 0).
template <int LAYOUT>
__device__ __forceinline__ void fp32_tile(const float* a, int64_t a_ld, const float* b, int64_t b_ld, int m0, int n0, int m, int n, int k0, int k1,
                                          float (&out)[4][4], float (&sums)[4]) {
  __shared__ __align__(16) float sa[DEPTH][TILE + 4], sb[DEPTH][TILE + 4];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4], part[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    sums[i] = part[i] = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = out[i][j] = 0.f;
  }
  int chain = 0;
  for (int k = k0; k < k1; k += DEPTH) {
#pragma unroll
    for (int i = threadIdx.x; i < TILE * DEPTH; i += FP32_THREADS) {
      {
        const int kk = LAYOUT == CLASSES_BY_ROWS ? i / TILE : i % DEPTH, r = LAYOUT == CLASSES_BY_ROWS ? i % TILE : i / DEPTH;
        const bool in = k + kk < k1 && m0 + r < m;
        sa[kk][r] = in ? __ldg(LAYOUT == CLASSES_BY_ROWS ? a + (int64_t)(k + kk) * a_ld + m0 + r : a + (int64_t)(m0 + r) * a_ld + k + kk) : 0.f;
      }
      {
        const int kk = LAYOUT == LOGITS ? i % DEPTH : i / TILE, r = LAYOUT == LOGITS ? i / DEPTH : i % TILE;
        const bool in = k + kk < k1 && n0 + r < n;
        sb[kk][r] = in ? __ldg(LAYOUT == LOGITS ? b + (int64_t)(n0 + r) * b_ld + k + kk : b + (int64_t)(k + kk) * b_ld + n0 + r) : 0.f;
      }
    }
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < DEPTH; ++kk) {
      const float4 u = *reinterpret_cast<const float4*>(&sa[kk][ty * 4]), v = *reinterpret_cast<const float4*>(&sb[kk][tx * 4]);
      const float x[4] = {u.x, u.y, u.z, u.w}, y[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        part[i] += x[i];
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(x[i], y[j], acc[i][j]);
      }
    }
    __syncthreads();
    if (++chain == CHAIN / DEPTH || k + DEPTH >= k1) {
      chain = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sums[i] += part[i];
        part[i] = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) { out[i][j] += acc[i][j]; acc[i][j] = 0.f; }
      }
    }
  }
}

}  // namespace
