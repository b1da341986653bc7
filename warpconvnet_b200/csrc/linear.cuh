// What the kernels of linear layers (linear.cu, linear_tcgen05.cu) share.
#pragma once
#include "philox.cuh"

enum wcn_linear_act { WCN_ACT_NONE = 0, WCN_ACT_RELU = 1, WCN_ACT_SILU = 2, WCN_ACT_GELU = 3 };
constexpr int WCN_E4M3 = 8;   // operands' type beside the WCN_* dtypes

// z[m][n] = sum over k of A[m][k] B[n][k] (or B[k][n]); with z + bias: out = add + dropout(act(z)); or, `grad`: out = dropout(add) act'(z).
struct wcn_linear_product {
  const void* a;
  const void* b;
  int64_t a_ld, b_ld;       // elements from row to row
  int m, n, k;
  const float* a_scale;     // of each row of A and of B (8 bits)
  const float* b_scale;
  void* out;                // [m][n], rows out_ld elements apart
  int64_t out_ld;
  const void* bias;         // [n] of the type of `out`; null: none
  int act;
  bool grad;
  const void* add;          // residual, or the result's gradient; null: none
  int64_t add_ld;
  wcn_drop drop;
  int64_t row0;             // place of the first row among all rows (for what is dropped)
  float factor;             // of dx (products of gradients alone)
};

// An fp32 matrix and where its parts go (linear_split_tcgen05.cu).
struct wcn_linear_matrix {
  const float* x;
  void* planes;
  int64_t rows, ld;
  int cols;
};
