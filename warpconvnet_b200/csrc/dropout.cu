// y = residual + keep x / (1 - p) of [n, channels] rows (the gradient is the same of dy): see philox.cuh for what is kept.
//
// Bound by HBM.  A thread has eight columns of a row, the elements of one call of the generator, and two such pieces at a time.
#include "philox.cuh"

namespace {

constexpr int THREADS = 256, PIECES = 2;

template <typename T> struct DropParams {
  const T* x;
  const T* residual;      // null: none
  T* y;                   // contiguous
  int64_t x_ld, res_ld, pieces;
  int c, across;          // columns, pieces of a row
  wcn_drop drop;
};

// Columns col .. of a row; WHOLE: eight of them in 16-byte loads.
template <typename T, bool WHOLE> __device__ __forceinline__ void load_eight_of(const T* row, int col, int c, T (&v)[8]) {
  if (WHOLE) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i)
      reinterpret_cast<uint4*>(v)[i] = __ldg(reinterpret_cast<const uint4*>(row + col) + i);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = col + i < c ? row[col + i] : wcn_from_float<T>(0.f);
  }
}

template <typename T, bool WHOLE>
__global__ void __launch_bounds__(THREADS) dropout_kernel(const __grid_constant__ DropParams<T> p) {
  const uint64_t seed = drop_seed(p.drop);
  const int64_t step = (int64_t)gridDim.x * THREADS;
  for (int64_t first = (int64_t)blockIdx.x * THREADS + threadIdx.x; first < p.pieces; first += PIECES * step) {
    __align__(16) T x[PIECES][8], r[PIECES][8];
    int64_t row[PIECES];
    int col[PIECES];
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
      const int64_t at = first + j * step;
      if (at >= p.pieces) continue;
      row[j] = at < (1ll << 32) ? (int64_t)((uint32_t)at / (uint32_t)p.across) : at / p.across;
      col[j] = (int)(at - row[j] * p.across) * 8;
      load_eight_of<T, WHOLE>(p.x + row[j] * p.x_ld, col[j], p.c, x[j]);
      if (p.residual) load_eight_of<T, WHOLE>(p.residual + row[j] * p.res_ld, col[j], p.c, r[j]);
    }
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
      if (first + j * step >= p.pieces) continue;
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = wcn_to_float<T>(x[j][i]);
      drop_eight(p.drop, seed, (uint32_t)col[j] / 8, (uint64_t)row[j], v);
      if (p.residual)
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += wcn_to_float<T>(r[j][i]);
      __align__(16) T out[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) out[i] = wcn_from_float<T>(v[i]);
      T* const y = p.y + row[j] * p.c + col[j];
      if (WHOLE) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(y)[i] = reinterpret_cast<const uint4*>(out)[i];
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (col[j] + i < p.c) y[i] = out[i];
      }
    }
  }
}

template <typename T>
int run_dropout(const void* x, int64_t x_ld, const void* residual, int64_t res_ld, int64_t n, int c, const wcn_drop& drop, void* y, cudaStream_t st) {
  DropParams<T> p = {(const T*)x, (const T*)residual, (T*)y, x_ld, res_ld, 0, c, (c + 7) / 8, drop};
  p.pieces = n * p.across;
  const int64_t e = sizeof(T);
  auto fits = [&](const void* at, int64_t ld) { return reinterpret_cast<uintptr_t>(at) % 16 == 0 && ld * e % 16 == 0; };
  const bool whole = c % 8 == 0 && fits(x, x_ld) && fits(y, c) && (!residual || fits(residual, res_ld));
  const int64_t blocks = (p.pieces + THREADS * PIECES - 1) / (THREADS * PIECES), most = 1 << 20;
  const unsigned grid = (unsigned)(blocks < most ? blocks : most);
  if (whole) dropout_kernel<T, true><<<grid, THREADS, 0, st>>>(p);
  else dropout_kernel<T, false><<<grid, THREADS, 0, st>>>(p);
  WCN_CHECK_LAUNCH();
  return WCN_OK;
}

}  // namespace

extern "C" int wcn_dropout(const void* x, int64_t x_ld, const void* residual, int64_t residual_ld, int64_t n, int32_t channels, int dtype,
                           int32_t least, int64_t seed, const int64_t* seed_at, void* y, void* stream) {
  if (n < 0 || channels <= 0 || least < 0 || least > 65536 || dtype < WCN_F32 || dtype > WCN_BF16) return WCN_ERR_INVALID_PARAMETERS;
  if (n == 0) return WCN_OK;
  if (!x || !y || (n > 1 && (x_ld < channels || (residual && residual_ld < channels)))) return WCN_ERR_INVALID_PARAMETERS;
  const wcn_drop drop = wcn_make_drop((uint32_t)least, seed, seed_at);
  cudaStream_t st = wcn_stream(stream);
  if (dtype == WCN_F32) return run_dropout<float>(x, x_ld, residual, residual_ld, n, channels, drop, y, st);
  if (dtype == WCN_F16) return run_dropout<__half>(x, x_ld, residual, residual_ld, n, channels, drop, y, st);
  return run_dropout<__nv_bfloat16>(x, x_ld, residual, residual_ld, n, channels, drop, y, st);
}
