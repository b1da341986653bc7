// Linear layers over rows, y = residual + dropout(act(x W^T + bias)) with x [n, k], W [m, k], and their gradients, with z = x W^T + bias:
//     dz = dropout'(dy) act'(z),   dx = dz W,   dW = dz^T x,   dbias = column sums of dz,   dresidual = dy.
//
// z is computed again in the backward pass, not kept: for rows as wide as these a product costs less than writing z and reading it (at
// 1.4 PFLOP/s and 6.5 TB/s up to some 400 inputs), and a training step holds x alone.  Gradients of narrow layers in 16 bits are one
// kernel's (linear_backward_tcgen05.cu).  Elsewhere dz, rounded to the inputs' type, goes to the workspace, in pieces of at most 512 MB (or 128 rows)
// (pieces that stay in L2 lost more by their launches than they gained: 240 000 x 96 -> 384 in pieces of 64 MB 241 us, whole 196); each
// is multiplied by W (dx) and by x (dW), whose sums over the rows are divided among the multiprocessors, in 16 bits into parts of
// 8192 rows at most too, and joined in a fixed order and in double: the same bits on every run.
//
// 16- and 8-bit operands run on the tensor cores (linear_tcgen05.cu; dW: the transposed product of linear_ce_tcgen05.cu), fp32 there too
// as sums of three bf16 numbers (linear_split_tcgen05.cu).  On the FMA pipes in tiles of 64 x 64 fp32 took as long for the smallest problems
// and up to four times as long for others (us forward, gradients: 500 x 64 -> 64 18, 51 and here 17, 35; 20 000 x 32 -> 32 16, 53 and 19,
// 40; 100 000 x 96 -> 200 251, 608 and 85, 174).
#include "linear.cuh"
#include "linear_ce.cuh"

int wcn_linear_run(const wcn_linear_product& q, int kind, bool bf16, bool by_k, int32_t* dev_status, cudaStream_t st);
int wcn_linear_backward_blocks(int64_t rows, int k, int n, int act, bool sums);
int wcn_linear_backward_run(const wcn_linear_product& q, float* slab, float* slab_ones, bool bf16, int32_t* dev_status, cudaStream_t st);
int wcn_dropout_rows(const void* x, int64_t x_ld, const void* residual, int64_t res_ld, int64_t n, int c, int dtype, const wcn_drop& drop, int64_t row0, void* y,
                     int64_t y_ld, cudaStream_t st);
int64_t wcn_linear_parts_bytes(int64_t rows, int cols);
int wcn_linear_parts(const wcn_linear_matrix* m, int count, cudaStream_t st);
int wcn_linear_split(const wcn_linear_product& q, bool by_k, const void* a_planes, const void* b_planes, int32_t* dev_status, cudaStream_t st);
int wcn_linear_split_weight(const wcn_ce_product& c, const void* a_planes, const void* b_planes, int32_t* dev_status, cudaStream_t st);
int wcn_linear_split_splits(int m, int n, int k);
int wcn_ce_product_splits(int m, int n, int k, bool blocked, bool ones);
int wcn_ce_product_run(const wcn_ce_product& q, bool transposed, bool blocked, int dtype, int32_t* dev_status, cudaStream_t st);

namespace {

constexpr int THREADS = 256;
constexpr int MOST_ROWS = 0x7FFE0000, MOST_INPUTS = 32768, MOST_OUTPUTS = 1 << 20;   // (row numbers, and some tiles behind the last, are 32-bit)
constexpr int64_t PIECE_BYTES = 512ll << 20;   // of dz
// Rows that an accumulator of a tensor core sums, at most (16 bits; dW and dbias).  It cuts what lies below its last place instead of
// rounding: sums of one sign lose 1.4e-7 of themselves for each 16 rows (dW of 1.2 million x 64 -> 64, 8 100 rows a block, came out
// 7e-5 short, of 10 million 2.4e-4, of 30 million 9e-4, where half a step of fp16 is 2.4e-4 at least).  With these, 7e-5.
constexpr int MOST_SUMMED = 8192;
// The same of the products that are one launch's, over inputs (which are not more) and over outputs (dx): 2 048 steps, 3e-4.
constexpr int MOST_TERMS = 32768;
static_assert(MOST_INPUTS <= MOST_TERMS, "sums over the inputs are not divided");

// ------------------------------------------------------------------ sums of the splits

struct JoinParams {
  const float* slab;        // [splits][m][ld]
  const float* ones;        // [splits][m]
  void* dw;                 // [m][n]; null: not wanted
  void* db;                 // [m]; null: not wanted
  int m, n, ld, splits;
  int quads;                // blocks for dw
  float factor;
  const int32_t* dev_status;
};

constexpr int SIDE = 8;     // threads that share the splits
template <typename T> __global__ void __launch_bounds__(THREADS) linear_join_kernel(const __grid_constant__ JoinParams p) {
  __shared__ double part[SIDE][THREADS / SIDE][4];
  const int side = threadIdx.x / (THREADS / SIDE), at = threadIdx.x % (THREADS / SIDE);
  const bool of_w = (int)blockIdx.x < p.quads;
  const int64_t all = of_w ? (int64_t)p.m * (p.ld / 4) : p.m, i = (int64_t)(of_w ? blockIdx.x : blockIdx.x - p.quads) * (THREADS / SIDE) + at;
  double v[4] = {0, 0, 0, 0};
  if (i < all) {
    if (of_w) {
#pragma unroll 4
      for (int s = side; s < p.splits; s += SIDE) {
        const float4 t = __ldg(reinterpret_cast<const float4*>(p.slab) + (int64_t)s * all + i);
        v[0] += t.x; v[1] += t.y; v[2] += t.z; v[3] += t.w;
      }
    } else {
#pragma unroll 4
      for (int s = side; s < p.splits; s += SIDE) v[0] += __ldg(&p.ones[(int64_t)s * all + i]);
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) part[side][at][j] = v[j];
  __syncthreads();
  if (side || i >= all) return;
  for (int s = 1; s < SIDE; ++s)
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] += part[s][at][j];
  const bool failed = *p.dev_status == (int)WCN_ERR_WAIT_EXPIRED;
  const float nan = __int_as_float(0x7FC00000);
  if (!of_w) {
    reinterpret_cast<T*>(p.db)[i] = wcn_from_float<T>(failed ? nan : (float)v[0] * p.factor);
    return;
  }
  const int64_t row = i / (p.ld / 4);
  const int col = (int)(i % (p.ld / 4)) * 4;
  T* const out = reinterpret_cast<T*>(p.dw) + row * p.n + col;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (col + j < p.n) out[j] = wcn_from_float<T>(failed ? nan : (float)v[j] * p.factor);
}

int join(JoinParams p, int dtype, cudaStream_t st) {
  constexpr int per = THREADS / SIDE;
  p.quads = p.dw ? (int)(((int64_t)p.m * (p.ld / 4) + per - 1) / per) : 0;
  const unsigned blocks = (unsigned)(p.quads + (p.db ? (p.m + per - 1) / per : 0));
  if (dtype == WCN_F32) linear_join_kernel<float><<<blocks, THREADS, 0, st>>>(p);
  else if (dtype == WCN_F16) linear_join_kernel<__half><<<blocks, THREADS, 0, st>>>(p);
  else linear_join_kernel<__nv_bfloat16><<<blocks, THREADS, 0, st>>>(p);
  ++wcn_launched;
  return cudaGetLastError() == cudaSuccess ? WCN_OK : WCN_ERR_EXECUTION;
}

// ------------------------------------------------------------------ plans

int run(const wcn_linear_product& q, int dtype, bool by_k, const void* a_planes, const void* b_planes, int32_t* dev_status, cudaStream_t st) {
  if (dtype != WCN_F32) return wcn_linear_run(q, dtype, dtype == WCN_BF16, by_k, dev_status, st);
  return wcn_linear_split(q, by_k, a_planes, b_planes, dev_status, st);
}
int weight_splits(int m, int k, int rows, int dtype, bool bias) {
  if (dtype == WCN_F32) return wcn_linear_split_splits(m, k, rows);   // (which adds its accumulators to sums in registers)
  const int splits = wcn_ce_product_splits(m, k, rows, false, bias), least = (int)(((int64_t)rows + MOST_SUMMED - 1) / MOST_SUMMED);
  return splits > least ? splits : least;
}

// The pieces of rows that dz is made in (forward: that x's parts are made in), and the workspace: dz of a piece, parts of x, dz and w, sums
// of dW and of dbias.
struct Pieces {
  int rows, count, splits, last_splits;   // of a piece; pieces; splits of a full piece and of the last one
  bool whole;                             // the kernel that makes all of them (16 bits, narrow layers); its splits are its blocks
  bool parts;                             // fp32: the operands are sums of three bf16 numbers
  int x_splits;                           // of dx: parts of the outputs (0: one launch finishes it)
  int64_t dz_ld, x_slab, x_parts, dz_parts, w_parts, slab, ones, bytes;
};
enum Want { DX = 1, DW = 2, DB = 4 };     // none of them: forward
// aligned: dy is read as x is (fp32 numbers always are).
Pieces plan(int64_t n, int k, int m, int dtype, int what, int act, bool drops, bool aligned) {
  Pieces p = {};
  aligned = aligned || dtype == WCN_F32;
  const int64_t e = wcn_dtype_size(dtype);
  const bool direct = aligned && act == WCN_ACT_NONE && !drops;
  auto round = [](int64_t v, int64_t to) { return (v + to - 1) / to * to; };
  if (what && dtype != WCN_F32) p.whole = wcn_linear_backward_blocks(n, k, m, act, what & DB) > 0;
  if (p.whole) {
    p.dz_ld = round(m, 8);
    int64_t most = (int64_t)wcn_num_sms() * MOST_SUMMED;
    if (!aligned && PIECE_BYTES / (p.dz_ld * e) < most) most = PIECE_BYTES / (p.dz_ld * e) / 128 * 128;   // (a copy of dy as the kernel reads it)
    const int64_t count = (n + most - 1) / most, rows = round((n + count - 1) / count, 128);
    p.rows = (int)(rows < n ? rows : n);
    p.count = (int)((n + p.rows - 1) / p.rows);
    p.splits = wcn_linear_backward_blocks(p.rows, k, m, act, what & DB);
    p.last_splits = wcn_linear_backward_blocks(n - (int64_t)(p.count - 1) * p.rows, k, m, act, what & DB);
    const int64_t all = (int64_t)p.splits * (p.count - 1) + p.last_splits;
    p.slab = aligned ? 0 : round(p.rows * p.dz_ld * e, 128);
    p.ones = p.slab + (what & (DW | DB) ? round(all * m * wcn_ce_round(k, 16) * 4, 128) : 0);
    p.bytes = p.ones + (what & DB ? all * m * 4 : 0);
    return p;
  }
  p.dz_ld = round(m, 16 / e);
  p.parts = dtype == WCN_F32;
  const bool weights = what & (DW | DB), makes_dz = what && !direct;
  const bool of_x = p.parts && (!what || makes_dz || weights), of_dz = p.parts && what, of_w = p.parts && (!what || makes_dz || (what & DX));
  if (what & DX && dtype != WCN_F32 && m > MOST_TERMS) p.x_splits = (m + MOST_TERMS - 1) / MOST_TERMS;
  const int64_t x_slab = (int64_t)p.x_splits * wcn_ce_round(k, 16) * 4;
  const int64_t each = x_slab + (makes_dz ? p.dz_ld * e : 0) + (of_x ? round(k, 8) * 6 : 0) + (of_dz ? round(m, 8) * 6 : 0);   // bytes of a row of a piece
  int64_t rows = each ? PIECE_BYTES / each / 128 * 128 : n;
  if (rows < 128) rows = 128;
  const int64_t count = (n + rows - 1) / rows;
  rows = round((n + count - 1) / count, 128);
  p.rows = (int)(rows < n ? rows : n);
  p.count = (int)((n + p.rows - 1) / p.rows);
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += round(bytes, 128);
    return here;
  };
  take(makes_dz ? p.rows * p.dz_ld * e : 0);
  p.x_slab = take(p.rows * x_slab);
  p.x_parts = take(of_x ? wcn_linear_parts_bytes(p.rows, k) : 0);
  p.dz_parts = take(of_dz ? wcn_linear_parts_bytes(p.rows, m) : 0);
  p.w_parts = take(of_w ? wcn_linear_parts_bytes(m, k) : 0);
  if (weights) {
    const int last = (int)(n - (int64_t)(p.count - 1) * p.rows);
    p.splits = weight_splits(m, k, p.rows, dtype, what & DB);
    p.last_splits = weight_splits(m, k, last, dtype, what & DB);
    const int64_t all = (int64_t)p.splits * (p.count - 1) + p.last_splits;
    p.slab = take(all * m * wcn_ce_round(k, 16) * 4);
    p.ones = take(what & DB ? all * m * 4 : 0);
  }
  p.bytes = at;
  return p;
}

bool sizes_taken(int64_t n, int k, int m) { return n >= 0 && n <= MOST_ROWS && k >= 1 && k <= MOST_INPUTS && m >= 1 && m <= MOST_OUTPUTS; }
bool rows_taken(const void* p, int64_t ld, int64_t rows, int columns, int size) {
  const int whole = size == 4 ? 1 : 16 / size;
  return p && reinterpret_cast<uintptr_t>(p) % (size == 4 ? 4 : 16) == 0 && ld % whole == 0 && (rows <= 1 || ld >= columns);
}

}  // namespace

extern "C" int wcn_linear(const void* x, int64_t x_ld, int64_t n, int32_t k, const void* w, int64_t w_ld, int32_t m, int dtype, const void* bias,
                          int act, const void* residual, int64_t residual_ld, int32_t least, int64_t seed, const int64_t* seed_at, void* y,
                          void* workspace, int64_t workspace_bytes, int32_t* dev_status, void* stream) {
  wcn_launched = 0;
  if (!sizes_taken(n, k, m) || dtype < WCN_F32 || dtype > WCN_BF16 || act < 0 || act > 3 || least < 0 || least > 65536) return WCN_ERR_INVALID_PARAMETERS;
  if (n == 0) return WCN_OK;
  const int size = wcn_dtype_size(dtype);
  if (!rows_taken(x, x_ld, n, k, size) || !rows_taken(w, w_ld, m, k, size) || !y || !dev_status || (residual && n > 1 && residual_ld < m))
    return WCN_ERR_INVALID_PARAMETERS;
  cudaStream_t st = wcn_stream(stream);
  wcn_linear_product q = {x, w, x_ld, w_ld, (int)n, m, k, nullptr, nullptr, y, m, bias, act, false, residual, residual_ld,
                          wcn_make_drop((uint32_t)least, seed, seed_at), 0};
  if (dtype != WCN_F32) return run(q, dtype, false, nullptr, nullptr, dev_status, st);
  const Pieces p = plan(n, k, m, dtype, 0, act, least, false);
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 31) || workspace_bytes < p.bytes) return WCN_ERR_INVALID_PARAMETERS;
  char* const ws = reinterpret_cast<char*>(workspace);
  for (int i = 0; i < p.count; ++i) {
    const int64_t r0 = (int64_t)i * p.rows;
    q.m = (int)(n - r0 < p.rows ? n - r0 : p.rows);
    q.a = (const float*)x + r0 * x_ld;
    q.out = (float*)y + r0 * m;
    q.add = residual ? (const float*)residual + r0 * residual_ld : nullptr;
    q.row0 = r0;
    const wcn_linear_matrix of[2] = {{(const float*)q.a, ws + p.x_parts, q.m, x_ld, k}, {(const float*)w, ws + p.w_parts, m, w_ld, k}};
    int rc = wcn_linear_parts(of, i ? 1 : 2, st);
    if (rc == WCN_OK) rc = run(q, dtype, false, ws + p.x_parts, ws + p.w_parts, dev_status, st);
    if (rc != WCN_OK) return rc;
  }
  return WCN_OK;
}

extern "C" int wcn_linear_8bit(const void* x, int64_t x_ld, const float* x_scale, int64_t n, int32_t k, const void* w, int64_t w_ld,
                               const float* w_scale, int32_t m, int out_dtype, const void* bias, int act, const void* residual,
                               int64_t residual_ld, void* y, int32_t* dev_status, void* stream) {
  wcn_launched = 0;
  if (!sizes_taken(n, k, m) || (out_dtype != WCN_F16 && out_dtype != WCN_BF16) || act < 0 || act > 3) return WCN_ERR_INVALID_PARAMETERS;
  if (n == 0) return WCN_OK;
  if (!rows_taken(x, x_ld, n, k, 1) || !rows_taken(w, w_ld, m, k, 1) || !x_scale || !w_scale || !y || !dev_status || (residual && n > 1 && residual_ld < m))
    return WCN_ERR_INVALID_PARAMETERS;
  wcn_linear_product q = {x, w, x_ld, w_ld, (int)n, m, k, x_scale, w_scale, y, m, bias, act, false, residual, residual_ld, wcn_make_drop(0, 0, nullptr), 0};
  return wcn_linear_run(q, WCN_E4M3, out_dtype == WCN_BF16, false, dev_status, wcn_stream(stream));
}

extern "C" int wcn_linear_workspace_bytes(int64_t n, int32_t k, int32_t m, int dtype, int32_t what, int act, int32_t least, int32_t aligned, int64_t* bytes) {
  if (!bytes || n < 1 || !sizes_taken(n, k, m) || dtype < WCN_F32 || dtype > WCN_BF16 || what < 0 || what > 7 || act < 0 || act > 3) return WCN_ERR_INVALID_PARAMETERS;
  *bytes = what || dtype == WCN_F32 ? plan(n, k, m, dtype, what, act, least != 0, aligned).bytes : 0;
  return WCN_OK;
}

extern "C" int wcn_linear_backward(const void* x, int64_t x_ld, int64_t n, int32_t k, const void* w, int64_t w_ld, int32_t m, int dtype,
                                   const void* bias, int act, const void* dy, int64_t dy_ld, int32_t least, int64_t seed, const int64_t* seed_at,
                                   void* dx, void* dw, void* db, void* workspace, int64_t workspace_bytes, int32_t* dev_status, void* stream) {
  wcn_launched = 0;
  if (!sizes_taken(n, k, m) || n == 0 || dtype < WCN_F32 || dtype > WCN_BF16 || act < 0 || act > 3 || least < 0 || least > 65536) return WCN_ERR_INVALID_PARAMETERS;
  const int size = wcn_dtype_size(dtype), what = (dx ? DX : 0) | (dw ? DW : 0) | (db ? DB : 0);
  // (rows of a gradient between boundaries are brought to them as others are made)
  const bool aligned = rows_taken(dy, dy_ld, n, m, size), direct = act == WCN_ACT_NONE && least == 0 && aligned;
  if (!what || !dev_status || !rows_taken(x, x_ld, n, k, size) || !rows_taken(w, w_ld, m, k, size) || !dy || reinterpret_cast<uintptr_t>(dy) % size ||
      (n > 1 && dy_ld < m))
    return WCN_ERR_INVALID_PARAMETERS;
  const Pieces p = plan(n, k, m, dtype, what, act, least != 0, aligned);
  if (p.bytes && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 31) || workspace_bytes < p.bytes)) return WCN_ERR_INVALID_PARAMETERS;
  char* const ws = reinterpret_cast<char*>(workspace);
  cudaStream_t st = wcn_stream(stream);
  const wcn_drop none = wcn_make_drop(0, 0, nullptr);
  wcn_drop drop = wcn_make_drop((uint32_t)least, seed, seed_at);
  float factor = 1.f;
  // In 16 bits dz is what is kept of dy (times the slope): the factor comes to the fp32 sums.  Without an activation nothing is rounded then; with
  // one, dz in fp16 does not pass the type's end for the factor's sake.
  if (least && dtype != WCN_F32) {
    factor = drop.scale;
    drop.scale = 1.f;
  }
  const int ld = wcn_ce_round(k, 16);
  char *const xs = p.parts ? ws + p.x_parts : nullptr, *const dzs = p.parts ? ws + p.dz_parts : nullptr, *const wsp = p.parts ? ws + p.w_parts : nullptr;
  for (int i = 0; i < p.count; ++i) {
    const int64_t r0 = (int64_t)i * p.rows;
    const int rows = (int)(n - r0 < p.rows ? n - r0 : p.rows);
    const char *const xp = (const char*)x + r0 * x_ld * size, *const dyp = (const char*)dy + r0 * dy_ld * size;
    const void* dz = direct ? (const void*)dyp : (const void*)ws;
    const int64_t dz_ld = direct ? dy_ld : p.dz_ld;
    int rc = WCN_OK;
    float *const slab = dw || db ? (float*)(ws + p.slab) + (int64_t)i * p.splits * m * ld : nullptr, *const ones = db ? (float*)(ws + p.ones) + (int64_t)i * p.splits * m : nullptr;
    if (p.whole) {
      if (!aligned) rc = wcn_dropout_rows(dyp, dy_ld, nullptr, 0, rows, m, dtype, none, r0, ws, p.dz_ld, st);
      const wcn_linear_product q = {xp, w, x_ld, w_ld, rows, m, k, nullptr, nullptr, dx ? (char*)dx + r0 * k * size : nullptr, k, bias, act, true, aligned ? dyp : ws,
                                    aligned ? dy_ld : p.dz_ld, drop, r0, factor};
      if (rc == WCN_OK) rc = wcn_linear_backward_run(q, slab, ones, dtype == WCN_BF16, dev_status, st);
      if (rc != WCN_OK) return rc;
      continue;
    }
    if (p.parts) {   // of what is there already
      wcn_linear_matrix of[3];
      int count = 0;
      if (!direct || dw || db) of[count++] = {(const float*)xp, xs, rows, x_ld, k};
      if (i == 0 && (!direct || dx)) of[count++] = {(const float*)w, wsp, m, w_ld, k};
      if (direct) of[count++] = {(const float*)dyp, dzs, rows, dy_ld, m};
      if (count) rc = wcn_linear_parts(of, count, st);
      if (rc != WCN_OK) return rc;
    }
    if (!direct) {
      wcn_linear_product q = {xp, w, x_ld, w_ld, rows, m, k, nullptr, nullptr, ws, p.dz_ld, bias, act, true, dyp, dy_ld, drop, r0};
      rc = act ? run(q, dtype, false, xs, wsp, dev_status, st) : wcn_dropout_rows(dyp, dy_ld, nullptr, 0, rows, m, dtype, drop, r0, ws, p.dz_ld, st);
      if (rc == WCN_OK && p.parts) {
        const wcn_linear_matrix of = {(const float*)ws, dzs, rows, p.dz_ld, m};
        rc = wcn_linear_parts(&of, 1, st);
      }
      if (rc != WCN_OK) return rc;
    }
    if (dx && p.x_splits) {
      wcn_ce_product q = {};
      q.a = dz; q.a_ld = dz_ld; q.b = w; q.b_ld = w_ld;
      q.m = rows; q.n = k; q.k = m;
      q.splits = p.x_splits;
      q.slab = (float*)(ws + p.x_slab);
      rc = wcn_ce_product_run(q, false, false, dtype, dev_status, st);
      if (rc == WCN_OK) rc = join({q.slab, nullptr, (char*)dx + r0 * k * size, nullptr, rows, k, ld, p.x_splits, 0, factor, dev_status}, dtype, st);
      if (rc != WCN_OK) return rc;
    } else if (dx) {
      wcn_linear_product q = {dz, w, dz_ld, w_ld, rows, k, m, nullptr, nullptr, (char*)dx + r0 * k * size, k, nullptr, WCN_ACT_NONE, false, nullptr, 0, none, 0, factor};
      rc = run(q, dtype, true, dzs, wsp, dev_status, st);
      if (rc != WCN_OK) return rc;
    }
    if (dw || db) {
      wcn_ce_product q = {};
      q.a = dz; q.a_ld = dz_ld; q.b = xp; q.b_ld = x_ld;
      q.m = m; q.n = k; q.k = rows;
      q.splits = i + 1 < p.count ? p.splits : p.last_splits;
      q.slab = slab;
      q.slab_ones = ones;
      rc = p.parts ? wcn_linear_split_weight(q, dzs, xs, dev_status, st) : wcn_ce_product_run(q, true, false, dtype, dev_status, st);
      if (rc != WCN_OK) return rc;
    }
  }
  if (!dw && !db) return WCN_OK;
  return join({(const float*)(ws + p.slab), (const float*)(ws + p.ones), dw, db, m, k, ld, p.splits * (p.count - 1) + p.last_splits, 0, factor, dev_status}, dtype, st);
}
