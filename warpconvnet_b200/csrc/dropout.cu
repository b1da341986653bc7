// y = residual + keep x / (1 - p) of [n, channels] rows (the gradient is the same of dy): see philox.cuh for what is kept.
//
// Bound by HBM.  A thread has eight columns of a row, the elements of one call of the generator, and two such pieces at a time.
// 240 000 x 384 bf16 83 us (369 MB at 4.4 TB/s), with residual 95 (553 MB at 5.8 TB/s): a thread loads its pieces, then draws for them, so
// that without a residual too few bytes are on their way.
#include "philox.cuh"

namespace {

constexpr int THREADS = 256, PIECES = 2;

template <typename T> struct DropParams {
  const T* x;
  const T* residual;      // null: none
  T* y;
  int64_t x_ld, res_ld, y_ld, n, row0, step_rows;
  int c, across, step;    // columns, pieces of a row; threads of the grid: step_rows rows of pieces and `step` pieces
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
  const PhiloxKeys keys = philox_keys(drop_seed(p.drop));
  const int64_t first = (int64_t)blockIdx.x * THREADS + threadIdx.x;
  int64_t row = first / p.across;
  int at = (int)(first - row * p.across);   // piece of the row
  while (row < p.n) {
    __align__(16) T x[PIECES][8], r[PIECES][8];
    int64_t rows[PIECES];
    int ats[PIECES];
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
      rows[j] = row;
      ats[j] = at;
      if (row < p.n) {
        load_eight_of<T, WHOLE>(p.x + row * p.x_ld, at * 8, p.c, x[j]);
        if (p.residual) load_eight_of<T, WHOLE>(p.residual + row * p.res_ld, at * 8, p.c, r[j]);
      }
      row += p.step_rows;                   // (a division a piece would be a sixth of the instructions)
      at += p.step;
      if (at >= p.across) { at -= p.across; ++row; }
    }
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
      if (rows[j] >= p.n) break;
      float2 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = make_float2(wcn_to_float<T>(x[j][2 * i]), wcn_to_float<T>(x[j][2 * i + 1]));
      if (p.drop.least) drop_eight(p.drop, keys, (uint32_t)ats[j], (uint64_t)(p.row0 + rows[j]), v);
      if (p.residual)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __fadd2_rn(v[i], make_float2(wcn_to_float<T>(r[j][2 * i]), wcn_to_float<T>(r[j][2 * i + 1])));
      __align__(16) T out[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) out[i] = wcn_from_float<T>(i & 1 ? v[i / 2].y : v[i / 2].x);
      T* const y = p.y + rows[j] * p.y_ld + ats[j] * 8;
      if (WHOLE) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(y)[i] = reinterpret_cast<const uint4*>(out)[i];
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (ats[j] * 8 + i < p.c) y[i] = out[i];
      }
    }
  }
}

template <typename T>
int run_dropout(const void* x, int64_t x_ld, const void* residual, int64_t res_ld, int64_t n, int c, const wcn_drop& drop, int64_t row0, void* y, int64_t y_ld,
                cudaStream_t st) {
  DropParams<T> p = {(const T*)x, (const T*)residual, (T*)y, x_ld, res_ld, y_ld, n, row0, 0, c, (c + 7) / 8, 0, drop};
  const int64_t e = sizeof(T);
  auto fits = [&](const void* at, int64_t ld) { return reinterpret_cast<uintptr_t>(at) % 16 == 0 && ld * e % 16 == 0; };
  const bool whole = c % 8 == 0 && fits(x, x_ld) && fits(y, y_ld) && (!residual || fits(residual, res_ld));
  const int64_t blocks = (n * p.across + THREADS * PIECES - 1) / (THREADS * PIECES), most = 16 * (int64_t)wcn_num_sms();
  const unsigned grid = (unsigned)(blocks < most ? blocks : most);
  const int64_t threads = (int64_t)grid * THREADS;
  p.step_rows = threads / p.across;
  p.step = (int)(threads % p.across);
  if (whole) dropout_kernel<T, true><<<grid, THREADS, 0, st>>>(p);
  else dropout_kernel<T, false><<<grid, THREADS, 0, st>>>(p);
  ++wcn_launched;
  return cudaGetLastError() == cudaSuccess ? WCN_OK : WCN_ERR_EXECUTION;
}

}  // namespace

// Rows row0 .. of a larger matrix.
int wcn_dropout_rows(const void* x, int64_t x_ld, const void* residual, int64_t res_ld, int64_t n, int c, int dtype, const wcn_drop& drop, int64_t row0, void* y,
                     int64_t y_ld, cudaStream_t st) {
  if (dtype == WCN_F32) return run_dropout<float>(x, x_ld, residual, res_ld, n, c, drop, row0, y, y_ld, st);
  if (dtype == WCN_F16) return run_dropout<__half>(x, x_ld, residual, res_ld, n, c, drop, row0, y, y_ld, st);
  return run_dropout<__nv_bfloat16>(x, x_ld, residual, res_ld, n, c, drop, row0, y, y_ld, st);
}

extern "C" int wcn_dropout(const void* x, int64_t x_ld, const void* residual, int64_t residual_ld, int64_t n, int32_t channels, int dtype,
                           int32_t least, int64_t seed, const int64_t* seed_at, void* y, void* stream) {
  if (n < 0 || channels <= 0 || least < 0 || least > 65536 || dtype < WCN_F32 || dtype > WCN_BF16) return WCN_ERR_INVALID_PARAMETERS;
  if (n == 0) return WCN_OK;
  if (!x || !y || (n > 1 && (x_ld < channels || (residual && residual_ld < channels)))) return WCN_ERR_INVALID_PARAMETERS;
  return wcn_dropout_rows(x, x_ld, residual, residual_ld, n, channels, dtype, wcn_make_drop((uint32_t)least, seed, seed_at), 0, y, channels, wcn_stream(stream));
}
