// What the kernels of the linear cross entropy (linear_ce.cu, linear_ce_tcgen05.cu) share.
#pragma once
#include "wcn_common.cuh"

// What a gradient is multiplied by as it is finished: *g / *count * factor (0 where no row counts); or, with `rows`, the gradient of
// each row's loss (0 of a row that does not count) * factor.
struct wcn_ce_scale {
  const float* g;
  const int32_t* count;   // null: 1
  float factor;
  const float* rows;      // null: one number for all
  const int64_t* labels;  // (with rows)
  int64_t ignore, classes;
};

#ifdef __CUDACC__
__device__ __forceinline__ float wcn_ce_factor(const wcn_ce_scale& s) {
  const int count = s.count ? *s.count : 1;
  return count ? *s.g / (float)count * s.factor : 0.f;
}
__device__ __forceinline__ float wcn_ce_row_factor(const wcn_ce_scale& s, int64_t row) {
  const int64_t y = __ldg(&s.labels[row]);
  return y != s.ignore && y >= 0 && y < s.classes ? __ldg(&s.rows[row]) * s.factor : 0.f;
}
#endif

// The logits of a piece of rows x classes, as they are used: sums of exponentials (forward) or gradients (backward).
struct wcn_ce_piece {
  const void* x;            // first row of the piece
  const void* w;            // first class
  int64_t x_ld, w_ld;
  int rows, classes, channels;
  const float* bias2;       // bias / ln 2 (fp32: bias) from the first class on, -inf from the last class to a multiple of 256; null: none
  // forward: [parts][rows] of (largest, sum of exp(z - largest)), z in units of ln 2 (fp32: as it is)
  float2* part;
  float* label_logits;      // of each row, where its label names a class (fp32)
  // backward
  const float* lse2;        // of the piece's rows, in the logits' units
  const float* loss;
  const int64_t* labels;
  const float* row_scale;   // gradient of each row's loss (null: 1), divided by *row_max (0: all of them are 0 or no numbers)
  const float* row_max;
  int64_t ignore, first_class, all_classes;
  void* g;                  // [rows][g_ld]
  int64_t g_ld;
};

// Where the forward pass leaves its results when all classes of a row are one tile's (linear_ce.cu does it otherwise).
struct wcn_ce_result {
  const void* bias;         // as given, of bias_dtype (null: none)
  int bias_dtype, reduction;
  float* bias2;             // [classes rounded up to 256, + 256]
  float* lse2;
  float* loss_rows;
  float* loss;              // null: none wanted
  int32_t* count;
  double* block_sums;       // [blocks]
  int32_t* block_counts;
  unsigned* counter;
};

// D[m][n] = sum over k of A[m][k] B[k][n]: the sums of each split of k, or the finished result.
struct wcn_ce_product {
  const void* a;            // [k][m] (transposed) or [m][k]
  const void* b;            // [k][n]
  int64_t a_ld, b_ld;
  int m, n, k;
  int splits;
  float* slab;              // [splits][m][n rounded up to 16]
  float* slab_ones;         // [splits][m]: the sums of A alone; null: not wanted
  void* out;                // [m][n]: written instead of the slab (one split)
  wcn_ce_scale scale;
};

__host__ __device__ static inline int wcn_ce_round(int64_t v, int to) { return (int)((v + to - 1) / to * to); }
