// Cross entropy of a linear layer's logits z = x w^T + b [n rows, v classes] against one label per row, without keeping z:
//     loss_i = log sum_j exp(z_ij) - z_iy                       over rows whose label is not `ignore`: mean, sum, or each
//     g = s_i (softmax(z_i) - onehot(y_i))      dx = g w      dw = g^T x      db = sums of g's columns
//
// Forward: one pass over tiles of z, of which each row keeps a running (largest, sum of exponentials); then eight lanes a row put
// the pieces of its classes together and take z_iy from a product of their own (in 16 bits, where the label's logit would cost the
// tiles a comparison each; fp32 tiles leave it: another order of its sum would be an error of the small losses).  Backward: z again,
// piece by piece of rows x classes; a piece's g goes to the workspace in x's type and is multiplied by w and by x from there.
// Products whose sums over k are divided, or that several pieces add to, are put together in fp32 in a fixed order: the same bits
// on every run.
// g is rounded to 16 bits as softmax - onehot, without the factor of a mean, which the results are multiplied by in fp32: labels'
// entries are the largest ones and keep 8 (11) bits whatever the number of rows.  (In fp16 it is raised by 2^14: a probability
// of 2^-28 is still a normal number.)  Weights of single rows, over the largest of them, are in g; not in that of dx in fp16, for
// which z and g are then made once more: 240 000 rows x 96 channels x 200 classes 194 us both ways, where bf16 takes 139.
//
// 16-bit types run on the tensor cores (linear_ce_tcgen05.cu); fp32 on the FMA pipes here, in tiles of 64 x 64, sums of 128
// products at a time.  20 000 rows x 64 channels x 40 classes fp32, forward and backward: 79 us on the device in eight launches of
// 2 to 20 us (the host's part makes that 150; 40 of a tile's 64 classes are used).  30 000 x 256 x 32 768 classes bf16 forward and
// backward: 1.92 to 2.29 ms as the power cap sets the clock, 0.9 to 1.05 PFLOP/s of products (logits twice, dx and dw).
#include "linear_ce.cuh"

int wcn_ce_logits_parts(int rows, int classes);
int wcn_ce_whole_blocks(int rows, int classes, int channels);
int wcn_ce_logits(const wcn_ce_piece& q, const wcn_ce_result* out, int dtype, bool gradient, float lift, int32_t* dev_status, cudaStream_t st);
int wcn_ce_head_blocks(int64_t rows, int channels, int classes, bool bias);
int wcn_ce_head(const wcn_ce_piece& q, const wcn_ce_scale& scale, void* dx, float* slab, float* slab_ones, int dtype, float lift,
                int32_t* dev_status, cudaStream_t st);
int wcn_ce_product_splits(int m, int n, int k, bool blocked, bool ones);
int wcn_ce_product_run(const wcn_ce_product& q, bool transposed, bool blocked, int dtype, int32_t* dev_status, cudaStream_t st);
bool wcn_ce_rows_taken(int channels);
void wcn_ce_rows_plan(int rows, int classes, int* chunk, int* slots);
int wcn_ce_rows(const wcn_ce_piece& q, float* slab, int dtype, float lift, int32_t* dev_status, cudaStream_t st);

namespace {

constexpr int THREADS = 256;
constexpr float LOG2E = 1.4426950408889634f;
constexpr double LN2 = 0.6931471805599453;
constexpr int64_t PIECE_BYTES = 512ll << 20;   // of g
constexpr int PIECE_ROWS = 148 * 128;

inline float lift_of(int dtype) { return dtype == WCN_F16 ? 14.f : 0.f; }

// ------------------------------------------------------------------ around the products

template <typename T>
__global__ void __launch_bounds__(THREADS) ce_bias_kernel(const T* bias, int64_t v, int64_t padded, float unit, float* bias2) {
  for (int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x; i < padded; i += (int64_t)gridDim.x * THREADS)
    bias2[i] = i < v ? wcn_to_float<T>(bias[i]) * unit : -INFINITY;
}

struct LossParams {
  const void* x;
  const void* w;
  int64_t x_ld, w_ld, n, v;
  int c, parts, reduction;
  const float* bias2;
  const int64_t* labels;
  int64_t ignore;
  const float2* part;      // [parts][n]
  float* lse2;
  float* loss_rows;        // (fp32: before that, the labels' logits)
  float* loss;
  int32_t* count;
  double* block_sums;      // [blocks]
  int32_t* block_counts;   // [blocks]
  unsigned* counter;
  int32_t* dev_status;
};

// The product of a row and its label's weights: eight lanes share it in pieces of 16 bytes.
template <typename T> __device__ __forceinline__ float share_of_dot(const T* x, const T* w, int c, int lane) {
  constexpr int N = 16 / (int)sizeof(T);
  float dot = 0.f;
  int i = lane * N;
#pragma unroll 4
  for (; i + N <= c; i += 8 * N) {
    __align__(16) T a[N], b[N];
    *reinterpret_cast<uint4*>(a) = __ldg(reinterpret_cast<const uint4*>(x + i));
    *reinterpret_cast<uint4*>(b) = __ldg(reinterpret_cast<const uint4*>(w + i));
#pragma unroll
    for (int k = 0; k < N; ++k) dot = fmaf(wcn_to_float<T>(a[k]), wcn_to_float<T>(b[k]), dot);
  }
  for (; i < c; ++i) dot = fmaf(wcn_to_float<T>(x[i]), wcn_to_float<T>(w[i]), dot);   // (one lane's, the last)
  return dot;
}

// Exponential and logarithm of logits as they are kept: of rows in 16 bits in units of ln 2, where an exponential is one
// instruction; of fp32 rows as they are, since each rounding of a logit in other units would be one of |z| 2^-24 of its probability.
template <typename T> __device__ __forceinline__ float exp_of(float z) { return sizeof(T) == 4 ? expf(z) : exp2f(z); }
template <typename T> __device__ __forceinline__ float log_of(float s) { return sizeof(T) == 4 ? logf(s) : log2f(s); }

// Eight lanes a row: its loss from the sums of its classes' pieces and its label's logit.
template <typename T>
__global__ void __launch_bounds__(THREADS) ce_loss_kernel(const __grid_constant__ LossParams p) {
  __shared__ double s_sum[THREADS / 32];
  __shared__ int s_count[THREADS / 32];
  __shared__ bool last;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l = lane & 7;
  const bool failed = *(volatile int32_t*)p.dev_status == (int)WCN_ERR_WAIT_EXPIRED;
  double total = 0;
  int counted = 0;
  bool bad = false;
  const int64_t step = (int64_t)gridDim.x * (THREADS / 8);
  int64_t r = (int64_t)blockIdx.x * (THREADS / 8) + threadIdx.x / 8;
  int64_t y = r < p.n ? __ldg(&p.labels[r]) : p.ignore;
  for (int64_t first = r - lane / 8; first < p.n; first += step, r += step) {   // (a warp's four rows)
    const int64_t ahead = r + step < p.n ? __ldg(&p.labels[r + step]) : p.ignore;
    const bool live = r < p.n, counts = live && y != p.ignore && y >= 0 && y < p.v;
    bad |= live && y != p.ignore && !counts;
    float dot = 0.f;   // (fp32: the label's logit, of one lane)
    if constexpr (sizeof(T) == 4) dot = counts && l == 0 ? p.loss_rows[r] : 0.f;
    else if (counts) dot = share_of_dot<T>(reinterpret_cast<const T*>(p.x) + r * p.x_ld, reinterpret_cast<const T*>(p.w) + y * p.w_ld, p.c, l);
    float top = -INFINITY, sum = 0.f;
    if (live)
#pragma unroll 4
      for (int i = l; i < p.parts; i += 8) {
        const float2 q = __ldg(&p.part[(int64_t)i * p.n + r]);
        const float now = fmaxf(top, q.x), by = now == -INFINITY ? 0.f : now;
        sum = sum * exp_of<T>(top - by) + q.y * exp_of<T>(q.x - by);
        top = now;
      }
#pragma unroll
    for (int o = 4; o; o >>= 1) {
      dot += __shfl_xor_sync(0xFFFFFFFFu, dot, o);
      const float t = __shfl_xor_sync(0xFFFFFFFFu, top, o), s = __shfl_xor_sync(0xFFFFFFFFu, sum, o);
      const float now = fmaxf(top, t), by = now == -INFINITY ? 0.f : now;
      sum = sum * exp_of<T>(top - by) + s * exp_of<T>(t - by);
      top = now;
    }
    const float more = log_of<T>(sum), lse2 = top + more;
    float loss = 0.f;
    if (counts) {
      // (a difference of logits, not of one and the log-sum-exp as it is rounded)
      if constexpr (sizeof(T) == 4) {
        loss = (top - dot) + more;
      } else {
        // The product is summed in another order than the tile's, and up to 2e-5 beside it: more than the loss of a row that is sure of
        // its class.  Where all exponentials but the largest come to less than a half, any other class is more than one below the
        // largest (in units of ln 2): a label that is not is the largest, whose logit is known.
        float z = p.bias2 ? fmaf(dot, LOG2E, __ldg(&p.bias2[y])) : dot * LOG2E;
        if (sum < 1.5f && top - z < 0.5f) z = top;
        loss = ((top - z) + more) * (float)LN2;
      }
      if (loss < 0.f) loss = 0.f;                       // (roundings of a probability of one)
    }
    if (failed) loss = __int_as_float(0x7FC00000);
    if (live && l == 0) {
      total += (double)loss;
      counted += counts;
      p.lse2[r] = lse2;
      p.loss_rows[r] = loss;
    }
    y = ahead;
  }
#pragma unroll
  for (int o = 16; o >= 8; o >>= 1) {
    total += __shfl_xor_sync(0xFFFFFFFFu, total, o);
    counted += __shfl_xor_sync(0xFFFFFFFFu, counted, o);
  }
  if (bad && l == 0) wcn_report_bounds(p.dev_status);
  if (!p.loss) return;
  if (lane == 0) { s_sum[warp] = total; s_count[warp] = counted; }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < THREADS / 32; ++i) { total += s_sum[i]; counted += s_count[i]; }
    p.block_sums[blockIdx.x] = total;
    p.block_counts[blockIdx.x] = counted;
    __threadfence();
    last = atomicAdd(p.counter, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  total = 0;
  counted = 0;
  for (int i = threadIdx.x; i < (int)gridDim.x; i += THREADS) {
    total += __ldcg(&p.block_sums[i]);
    counted += __ldcg(&p.block_counts[i]);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    total += __shfl_xor_sync(0xFFFFFFFFu, total, o);
    counted += __shfl_xor_sync(0xFFFFFFFFu, counted, o);
  }
  if (lane == 0) { s_sum[warp] = total; s_count[warp] = counted; }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < THREADS / 32; ++i) { total += s_sum[i]; counted += s_count[i]; }
    *p.loss = (float)(p.reduction == 1 ? total / (double)counted : total);
    *p.count = counted;
    *p.counter = 0;
  }
}

// acc (+)= sums of the splits, or the finished result.  Four columns a thread, SIDE threads that share the splits.
struct JoinParams {
  const float* slab;       // [splits][m][ld]
  float* acc;              // [m][ld] (null: nothing before, nothing after)
  bool add;                // acc has something already
  void* out;               // [m][n]; null: acc is written
  int64_t m;
  int n, ld, splits;
  wcn_ce_scale scale;
  const int32_t* dev_status;
  int n_tiles, chunk;      // splits of a row as ce_rows_kernel leaves them (chunk 0: `splits` for all)
};

template <typename TO, int SIDE> __device__ __forceinline__ void join_quads(const JoinParams& p) {
  constexpr int QUADS = THREADS / SIDE;
  __shared__ double part[SIDE > 1 ? THREADS : 1][4];
  const int side = threadIdx.x / QUADS, at = threadIdx.x % QUADS;
  const int quads = p.ld / 4;
  const int64_t all = p.m * quads, q = (int64_t)blockIdx.x * QUADS + at;
  double v[4] = {0, 0, 0, 0};
  if (q < all) {
    const float4* const from = reinterpret_cast<const float4*>(p.slab) + q;
    int splits = p.splits;
    if (p.chunk) {
      const int64_t first = q / quads / 128 * p.n_tiles;
      splits = (int)((first + p.n_tiles - 1) / p.chunk - first / p.chunk) + 1;
    }
#pragma unroll 4
    for (int s = side; s < splits; s += SIDE) {
      const float4 t = __ldg(from + (int64_t)s * all);
      v[0] += t.x; v[1] += t.y; v[2] += t.z; v[3] += t.w;
    }
  }
  if (SIDE > 1) {
#pragma unroll
    for (int i = 0; i < 4; ++i) part[threadIdx.x][i] = v[i];
    __syncthreads();
    if (side) return;
    for (int s = 1; s < SIDE; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] += part[s * QUADS + at][i];
  }
  if (q >= all) return;
  const int64_t row = q / quads;
  const int col = (int)(q % quads) * 4;
  if (p.add) {
    const float4 t = reinterpret_cast<const float4*>(p.acc)[q];
    v[0] += t.x; v[1] += t.y; v[2] += t.z; v[3] += t.w;
  }
  if (!p.out) {
    reinterpret_cast<float4*>(p.acc)[q] = make_float4((float)v[0], (float)v[1], (float)v[2], (float)v[3]);
    return;
  }
  float scale = p.scale.rows ? wcn_ce_row_factor(p.scale, row) : wcn_ce_factor(p.scale);
  if (*p.dev_status == (int)WCN_ERR_WAIT_EXPIRED) scale = __int_as_float(0x7FC00000);
  TO* const out = reinterpret_cast<TO*>(p.out) + row * p.n + col;
  __align__(16) TO r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = wcn_from_float<TO>((float)v[i] * scale);
  if (p.n % 4 == 0) {   // (the result is a tensor's memory: its rows of whole quads start on their boundaries)
    if (col < p.n) {
      if (sizeof(TO) == 2) *reinterpret_cast<uint2*>(out) = *reinterpret_cast<const uint2*>(r);
      else *reinterpret_cast<uint4*>(out) = *reinterpret_cast<const uint4*>(r);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (col + i < p.n) out[i] = r[i];
  }
}

template <typename TO, int SIDE>
__global__ void __launch_bounds__(THREADS) ce_join_kernel(const __grid_constant__ JoinParams p) { join_quads<TO, SIDE>(p); }

// The same of one number a class: 32 classes a block, eight threads that share the splits.
template <typename TO>
__device__ __forceinline__ void join_sums(const JoinParams& p, int block) {
  __shared__ double part[THREADS / 32][33];
  const int lane = threadIdx.x & 31, side = threadIdx.x >> 5;
  const int64_t i = (int64_t)block * 32 + lane;
  double v = 0;
  if (i < p.m)
#pragma unroll 4
    for (int s = side; s < p.splits; s += THREADS / 32) v += (double)__ldg(&p.slab[(int64_t)s * p.m + i]);
  part[side][lane] = v;
  __syncthreads();
  if (side || i >= p.m) return;
  for (int s = 1; s < THREADS / 32; ++s) v += part[s][lane];
  if (p.add) v += (double)p.acc[i];
  if (!p.out) {
    p.acc[i] = (float)v;
    return;
  }
  float scale = wcn_ce_factor(p.scale);
  if (*p.dev_status == (int)WCN_ERR_WAIT_EXPIRED) scale = __int_as_float(0x7FC00000);
  reinterpret_cast<TO*>(p.out)[i] = wcn_from_float<TO>((float)v * scale);
}

template <typename TO>
__global__ void __launch_bounds__(THREADS) ce_join_sums_kernel(const __grid_constant__ JoinParams p) { join_sums<TO>(p, blockIdx.x); }

// Both of a small head in one launch: the blocks behind the first `blocks` do the second one's.
template <typename TO>
__global__ void __launch_bounds__(THREADS) ce_join_both_kernel(const __grid_constant__ JoinParams p, const __grid_constant__ JoinParams sums, int blocks) {
  if ((int)blockIdx.x < blocks) join_quads<TO, 8>(p);
  else join_sums<TO>(sums, blockIdx.x - blocks);
}

template <typename TO> int join_as(const JoinParams& p, cudaStream_t st) {
  ++wcn_launched;
  if (p.ld == 1) {
    ce_join_sums_kernel<TO><<<(unsigned)((p.m + 31) / 32), THREADS, 0, st>>>(p);
    return cudaGetLastError() == cudaSuccess ? WCN_OK : WCN_ERR_EXECUTION;
  }
  const int64_t all = p.m * (p.ld / 4);
  if (p.splits >= 16) ce_join_kernel<TO, 8><<<(unsigned)((all + THREADS / 8 - 1) / (THREADS / 8)), THREADS, 0, st>>>(p);
  else ce_join_kernel<TO, 1><<<(unsigned)((all + THREADS - 1) / THREADS), THREADS, 0, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? WCN_OK : WCN_ERR_EXECUTION;
}
int join(const JoinParams& p, int dtype, cudaStream_t st) {
  if (dtype == WCN_F32) return join_as<float>(p, st);
  if (dtype == WCN_F16) return join_as<__half>(p, st);
  return join_as<__nv_bfloat16>(p, st);
}

template <typename TO> int join_both_as(const JoinParams& p, const JoinParams& sums, cudaStream_t st) {
  const int blocks = (int)((p.m * (p.ld / 4) + THREADS / 8 - 1) / (THREADS / 8));
  ce_join_both_kernel<TO><<<(unsigned)(blocks + (sums.m + 31) / 32), THREADS, 0, st>>>(p, sums, blocks);
  ++wcn_launched;
  return cudaGetLastError() == cudaSuccess ? WCN_OK : WCN_ERR_EXECUTION;
}
int join_both(const JoinParams& p, const JoinParams& sums, int dtype, cudaStream_t st) {
  return dtype == WCN_F16 ? join_both_as<__half>(p, sums, st) : dtype == WCN_F32 ? join_both_as<float>(p, sums, st) : join_both_as<__nv_bfloat16>(p, sums, st);
}

// ------------------------------------------------------------------ fp32

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
    for (int i = threadIdx.x; i < TILE * DEPTH; i += THREADS) {
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

// A block has `per` tiles of classes side by side (GRAD: one), of which each row leaves one (largest, sum).
template <bool GRAD>
__global__ void __launch_bounds__(THREADS, 4) ce_logits_fp32_kernel(const __grid_constant__ wcn_ce_piece q, int per) {
  const int m0 = blockIdx.x * TILE, tx = threadIdx.x & 15, ty = threadIdx.x >> 4, n_tiles = (q.classes + TILE - 1) / TILE;
  __shared__ float2 so_far[TILE];   // of each row, its first thread's alone
  if (!GRAD && threadIdx.x < TILE) so_far[threadIdx.x] = make_float2(-INFINITY, 0.f);   // (barriers follow)
  for (int n = GRAD ? blockIdx.y : blockIdx.y * per, last = GRAD ? n + 1 : min(n + per, n_tiles); n < last; ++n) {
    const int n0 = n * TILE;
    float z[4][4], unused[4];
    fp32_tile<LOGITS>((const float*)q.x, q.x_ld, (const float*)q.w, q.w_ld, m0, n0, q.rows, q.classes, 0, q.channels, z, unused);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int col = n0 + tx * 4 + j;
        z[i][j] = col >= q.classes ? -INFINITY : q.bias2 ? z[i][j] + __ldg(&q.bias2[col]) : z[i][j];
      }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = m0 + ty * 4 + i;
      if (!GRAD) {
        if (row < q.rows) {
          const int64_t in = __ldg(&q.labels[row]) - (n0 + tx * 4);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (in == j && n0 + tx * 4 + j < q.classes) q.label_logits[row] = z[i][j];
        }
        float top = fmaxf(fmaxf(z[i][0], z[i][1]), fmaxf(z[i][2], z[i][3])), by = top == -INFINITY ? 0.f : top, sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) sum += expf(z[i][j] - by);
#pragma unroll
        for (int o = 8; o; o >>= 1) {   // the 16 threads of a row
          const float t = __shfl_xor_sync(0xFFFFFFFFu, top, o), s = __shfl_xor_sync(0xFFFFFFFFu, sum, o);
          const float now = fmaxf(top, t);
          by = now == -INFINITY ? 0.f : now;
          sum = sum * expf(top - by) + s * expf(t - by);
          top = now;
        }
        if (tx == 0) {
          const float2 old = so_far[ty * 4 + i];
          const float now = fmaxf(old.x, top);
          by = now == -INFINITY ? 0.f : now;
          so_far[ty * 4 + i] = make_float2(now, old.y * expf(old.x - by) + sum * expf(top - by));
        }
      } else if (row < q.rows) {
        const int64_t y = __ldg(&q.labels[row]);
        const bool counts = y != q.ignore && y >= 0 && y < q.all_classes;
        float scale = 1.f;
        if (q.row_scale) {
          const float most = __ldg(q.row_max);
          scale = __ldg(&q.row_scale[row]) / (most > 0.f ? most : 1.f);
        }
        const float lse = __ldg(&q.lse2[row]), loss = __ldg(&q.loss[row]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int col = n0 + tx * 4 + j;
          if (col >= q.classes) continue;
          float g = 0.f;
          if (counts) g = scale * (y - q.first_class == col ? expm1f(-loss) : expf(z[i][j] - lse));
          reinterpret_cast<float*>(q.g)[(int64_t)row * q.g_ld + col] = g;
        }
      }
    }
  }
  if (GRAD || tx) return;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (m0 + ty * 4 + i < q.rows) q.part[(int64_t)blockIdx.y * q.rows + m0 + ty * 4 + i] = so_far[ty * 4 + i];
}

template <bool TRANS>
__global__ void __launch_bounds__(THREADS) ce_product_fp32_kernel(const __grid_constant__ wcn_ce_product q, int per) {
  const int m0 = blockIdx.x * TILE, n0 = blockIdx.y * TILE, split = blockIdx.z, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float d[4][4], sums[4];
  const int k0 = split * per, k1 = min(k0 + per, q.k);
  fp32_tile<TRANS ? CLASSES_BY_ROWS : ROWS_BY_CLASSES>((const float*)q.a, q.a_ld, (const float*)q.b, q.b_ld, m0, n0, q.m, q.n, k0, k1, d, sums);
  const int ld = wcn_ce_round(q.n, 16);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = m0 + ty * 4 + i;
    if (row >= q.m) continue;
    if (n0 + tx * 4 < ld)
      *reinterpret_cast<float4*>(q.slab + ((int64_t)split * q.m + row) * ld + n0 + tx * 4) = make_float4(d[i][0], d[i][1], d[i][2], d[i][3]);
    if (q.slab_ones && n0 == 0 && tx == 0) q.slab_ones[(int64_t)split * q.m + row] = sums[i];
  }
}

int fp32_splits(int m, int n, int k) {
  const int64_t tiles = (int64_t)((m + TILE - 1) / TILE) * ((n + TILE - 1) / TILE), want = (8 * (int64_t)wcn_num_sms() + tiles - 1) / tiles;
  const int chains = (k + CHAIN - 1) / CHAIN;
  const int s = (int)(want < chains ? want : chains), per = (chains + s - 1) / s;
  return (chains + per - 1) / per;
}

int fp32_product(const wcn_ce_product& q, bool transposed, cudaStream_t st) {
  const int chains = (q.k + CHAIN - 1) / CHAIN, per = (chains + q.splits - 1) / q.splits * CHAIN;
  const dim3 grid((q.m + TILE - 1) / TILE, (q.n + TILE - 1) / TILE, q.splits);
  if (transposed) ce_product_fp32_kernel<true><<<grid, THREADS, 0, st>>>(q, per);
  else ce_product_fp32_kernel<false><<<grid, THREADS, 0, st>>>(q, per);
  ++wcn_launched;
  return cudaGetLastError() == cudaSuccess ? WCN_OK : WCN_ERR_EXECUTION;
}

// ------------------------------------------------------------------ plans

// Tiles of a block of fp32 losses: a row has at most 256 (largest, sum), 2 KB, as in 16 bits.
int tiles_a_part(int64_t v) { return (int)((v + 256 * TILE - 1) / (256 * TILE)); }

int logit_parts(int64_t n, int64_t v, int dtype) {
  const int64_t part = (int64_t)TILE * tiles_a_part(v);
  return dtype == WCN_F32 ? (int)((v + part - 1) / part) : wcn_ce_logits_parts((int)n, (int)v);
}
int loss_blocks(int64_t n) {
  const int64_t want = (n + THREADS / 8 - 1) / (THREADS / 8), most = 8 * (int64_t)wcn_num_sms();
  return (int)(want < most ? want : most);
}
int product_splits(int m, int n, int k, int dtype, bool blocked = false, bool ones = false) {
  return dtype == WCN_F32 ? fp32_splits(m, n, k) : wcn_ce_product_splits(m, n, k, blocked, ones);
}

// How the gradient of the logits is cut into pieces, and where everything is in the workspace.
struct Pieces {
  int64_t n, v;
  int c, ld, dtype;
  int rows, classes, row_pieces, class_pieces;
  int64_t g, slab_x, slab_w, slab_b, acc_x, acc_w, acc_b, bytes;
  int64_t g_ld;
  bool fused;            // g and dx are one kernel's
  int head;              // blocks of the kernel that needs no pieces (few classes), 0: not taken
};

int64_t aligned(int64_t bytes) { return (bytes + 255) / 256 * 256; }

Pieces cut(int64_t n, int c, int64_t v, int dtype, bool x, bool w, bool b) {
  Pieces p = {};
  p.n = n; p.v = v; p.c = c; p.dtype = dtype;
  p.ld = wcn_ce_round(c, 16);
  const int e = wcn_dtype_size(dtype);
  int64_t at = 0;
  auto take = [&](int64_t bytes) { const int64_t here = at; at += aligned(bytes); return here; };
  p.head = dtype != WCN_F32 && v <= 256 ? wcn_ce_head_blocks(n, c, (int)v, b) : 0;
  if (p.head) {
    p.slab_w = take(w || b ? (int64_t)p.head * v * p.ld * 4 : 0);
    p.slab_b = take(b ? (int64_t)p.head * v * 4 : 0);
    p.bytes = at;
    return p;
  }
  p.fused = dtype != WCN_F32 && v > 256 && wcn_ce_rows_taken(c);
  p.row_pieces = (int)((n + PIECE_ROWS - 1) / PIECE_ROWS);
  if (v <= 1024 || p.fused) {   // as many rows as there is room for with all classes or a good many
    const int64_t few = v <= 1024 ? (v + 63) / 64 * 64 : 1024, most = PIECE_BYTES / (e * few) / 128 * 128;
    p.row_pieces = (int)((n + most - 1) / most);
  }
  p.rows = wcn_ce_round((n + p.row_pieces - 1) / p.row_pieces, 128);
  p.row_pieces = (int)((n + p.rows - 1) / p.rows);
  if (p.rows > n) p.rows = (int)n;
  int64_t most = PIECE_BYTES / ((int64_t)(p.fused ? wcn_ce_round(p.rows, 128) : p.rows) * e) / 256 * 256;   // (fused: whole tiles of g)
  if (most < 1024) most = 1024;
  if (dtype == WCN_F32 && most > 65535 / 4 * 4 * TILE) most = 65535 / 4 * 4 * TILE;   // (a grid has 65 535 tiles in y)
  p.class_pieces = (int)((v + most - 1) / most);
  p.classes = p.class_pieces == 1 ? (int)v : wcn_ce_round((v + p.class_pieces - 1) / p.class_pieces, 256);
  p.class_pieces = (int)((v + p.classes - 1) / p.classes);
  p.g_ld = wcn_ce_round(p.classes, 64);
  // the largest slabs of any piece (the last ones are smaller, and their sums divided otherwise)
  int64_t sx = 0, sw = 0, sb = 0;
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < 2; ++j) {
      const int64_t r = i ? n - (int64_t)(p.row_pieces - 1) * p.rows : p.rows, k = j ? v - (int64_t)(p.class_pieces - 1) * p.classes : p.classes;
      int chunk, slots;
      if (p.fused) wcn_ce_rows_plan((int)r, (int)k, &chunk, &slots);
      else slots = product_splits((int)r, c, (int)k, dtype);
      const int64_t fx = slots * r * p.ld * 4, s = product_splits((int)k, c, (int)r, dtype, p.fused, b);
      if (fx > sx) sx = fx;
      if (s * k * p.ld * 4 > sw) sw = s * k * p.ld * 4;
      if (s * k * 4 > sb) sb = s * k * 4;
    }
  p.g = take(p.fused ? (w || b ? (int64_t)wcn_ce_round(p.rows, 128) * wcn_ce_round(p.classes, 128) * e : 0) : (int64_t)p.rows * p.g_ld * e);
  p.slab_x = take(x ? sx : 0);
  p.slab_w = take(w || b ? sw : 0);
  p.slab_b = take(b ? (sb + 15) / 16 * 16 : 0);
  p.acc_x = take(x && p.class_pieces > 1 ? (int64_t)p.rows * p.ld * 4 : 0);
  p.acc_w = take(w && p.row_pieces > 1 ? v * p.ld * 4 : 0);
  p.acc_b = take(b && p.row_pieces > 1 ? (v + 16) * 4 : 0);
  p.bytes = at;
  return p;
}

bool sizes_ok(int64_t n, int32_t c, int64_t v, int dtype) {
  return n > 0 && n < 0x7FFFFF00ll && v > 0 && v < 0x7FFFFF00ll && c > 0 && c <= 32768 && dtype >= WCN_F32 && dtype <= WCN_BF16;
}

bool matrix_ok(const void* p, int64_t ld, int c, int dtype) {
  if (!p || ld < c) return false;
  return dtype == WCN_F32 ? reinterpret_cast<uintptr_t>(p) % 4 == 0 : reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0;
}

bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool on32(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 31) == 0; }   // (what is written in pieces of 32 bytes)

}  // namespace

extern "C" int wcn_linear_ce_workspace_bytes(int64_t n, int32_t channels, int64_t classes, int dtype, int what, int64_t* bytes) {
  if (!bytes || !sizes_ok(n, channels, classes, dtype)) return WCN_ERR_INVALID_PARAMETERS;
  if (what) *bytes = cut(n, channels, classes, dtype, what & 1, what & 2, what & 4).bytes + 256;   // (never none)
  else *bytes = aligned((int64_t)logit_parts(n, classes, dtype) * n * 8) + (int64_t)loss_blocks(n) * 16;
  return WCN_OK;
}

extern "C" int wcn_linear_ce(const void* x, int64_t x_ld, int64_t n, int32_t channels, const void* w, int64_t w_ld, int64_t classes,
                             const void* bias, int bias_dtype, const int64_t* labels, int64_t ignore, int dtype, int reduction,
                             float* lse2, float* loss_rows, float* bias2, int32_t* count, float* loss, void* workspace,
                             int64_t workspace_bytes, uint32_t* counter, int32_t* dev_status, void* stream) {
  wcn_launched = 0;
  if (!sizes_ok(n, channels, classes, dtype) || !matrix_ok(x, x_ld, channels, dtype) || !matrix_ok(w, w_ld, channels, dtype) || !labels ||
      !lse2 || !loss_rows || !workspace || !on16(workspace) || !counter || !dev_status || (bias && (!bias2 || !on16(bias2))) ||
      reduction < 0 || reduction > 2 || (reduction && (!loss || !count)) || bias_dtype < WCN_F32 || bias_dtype > WCN_BF16)
    return WCN_ERR_INVALID_PARAMETERS;
  int64_t need = 0;
  wcn_linear_ce_workspace_bytes(n, channels, classes, dtype, 0, &need);
  if (need > workspace_bytes) return WCN_ERR_SCRATCH_TOO_SMALL;
  cudaStream_t st = wcn_stream(stream);
  if (const int blocks = dtype == WCN_F32 || classes > 256 ? 0 : wcn_ce_whole_blocks((int)n, (int)classes, channels)) {
    wcn_ce_piece q = {};
    q.x = x; q.w = w; q.x_ld = x_ld; q.w_ld = w_ld; q.rows = (int)n; q.classes = (int)classes; q.channels = channels;
    q.labels = labels; q.ignore = ignore; q.all_classes = classes;
    double* const sums = (double*)workspace;
    const wcn_ce_result out = {bias, bias_dtype, reduction, bias2, lse2, loss_rows, reduction ? loss : nullptr, count, sums, (int32_t*)(sums + blocks), counter};
    return wcn_ce_logits(q, &out, dtype, false, 0.f, dev_status, st);
  }
  if (bias) {
    const int64_t padded = (classes + 255) / 256 * 256 + 256;
    const unsigned blocks = (unsigned)((padded + THREADS - 1) / THREADS < 1024 ? (padded + THREADS - 1) / THREADS : 1024);
    const float unit = dtype == WCN_F32 ? 1.f : LOG2E;
    if (bias_dtype == WCN_F32) ce_bias_kernel<float><<<blocks, THREADS, 0, st>>>((const float*)bias, classes, padded, unit, bias2);
    else if (bias_dtype == WCN_F16) ce_bias_kernel<__half><<<blocks, THREADS, 0, st>>>((const __half*)bias, classes, padded, unit, bias2);
    else ce_bias_kernel<__nv_bfloat16><<<blocks, THREADS, 0, st>>>((const __nv_bfloat16*)bias, classes, padded, unit, bias2);
    ++wcn_launched;
  }
  const int parts = logit_parts(n, classes, dtype);
  wcn_ce_piece q = {};
  q.x = x; q.w = w; q.x_ld = x_ld; q.w_ld = w_ld; q.rows = (int)n; q.classes = (int)classes; q.channels = channels;
  q.bias2 = bias ? bias2 : nullptr;
  q.part = (float2*)workspace;
  q.labels = labels; q.ignore = ignore; q.all_classes = classes;
  q.label_logits = loss_rows;
  if (dtype == WCN_F32) {
    ce_logits_fp32_kernel<false><<<dim3((unsigned)((n + TILE - 1) / TILE), (unsigned)parts), THREADS, 0, st>>>(q, tiles_a_part(classes));
    ++wcn_launched;
  } else {
    const int rc = wcn_ce_logits(q, nullptr, dtype, false, 0.f, dev_status, st);
    if (rc != WCN_OK) return rc;
  }
  LossParams p = {};
  p.x = x; p.w = w; p.x_ld = x_ld; p.w_ld = w_ld; p.n = n; p.v = classes; p.c = channels; p.parts = parts; p.reduction = reduction;
  p.bias2 = q.bias2; p.labels = labels; p.ignore = ignore; p.part = q.part; p.lse2 = lse2; p.loss_rows = loss_rows;
  p.loss = reduction ? loss : nullptr; p.count = count; p.counter = counter; p.dev_status = dev_status;
  const int blocks = loss_blocks(n);
  p.block_sums = (double*)((char*)workspace + aligned((int64_t)parts * n * 8));
  p.block_counts = (int32_t*)(p.block_sums + blocks);
  if (dtype == WCN_F16) ce_loss_kernel<__half><<<blocks, THREADS, 0, st>>>(p);
  else if (dtype == WCN_BF16) ce_loss_kernel<__nv_bfloat16><<<blocks, THREADS, 0, st>>>(p);
  else ce_loss_kernel<float><<<blocks, THREADS, 0, st>>>(p);
  ++wcn_launched;
  return cudaGetLastError() == cudaSuccess ? WCN_OK : WCN_ERR_EXECUTION;
}

extern "C" int wcn_linear_ce_backward(const void* x, int64_t x_ld, int64_t n, int32_t channels, const void* w, int64_t w_ld,
                                      int64_t classes, const float* bias2, const int64_t* labels, int64_t ignore, int dtype,
                                      const float* lse2, const float* loss_rows, const int32_t* count, const float* grad,
                                      const float* row_max, void* dx, void* dw, void* dbias, int bias_dtype, void* workspace,
                                      int64_t workspace_bytes, int32_t* dev_status, void* stream) {
  wcn_launched = 0;
  if (!sizes_ok(n, channels, classes, dtype) || !matrix_ok(x, x_ld, channels, dtype) || !matrix_ok(w, w_ld, channels, dtype) || !labels ||
      !lse2 || !loss_rows || !grad || !workspace || !on32(workspace) || !on16(dx) || !on16(dw) || !dev_status || bias_dtype < WCN_F32 ||
      bias_dtype > WCN_BF16)
    return WCN_ERR_INVALID_PARAMETERS;
  if (!dx && !dw && !dbias) return WCN_OK;
  // Rows of their own weight in fp16: g of a row times its weight over the largest one would be subnormal where that is below 2^-28.
  // dx takes the weights in fp32 at its end, from a g without them; dw and dbias, which add rows up, from a g with them.
  const bool late = row_max && dtype == WCN_F16 && dx;
  if (late && (dw || dbias)) {
    const int rc = wcn_linear_ce_backward(x, x_ld, n, channels, w, w_ld, classes, bias2, labels, ignore, dtype, lse2, loss_rows, count, grad, row_max, nullptr,
                                          dw, dbias, bias_dtype, workspace, workspace_bytes, dev_status, stream);
    if (rc != WCN_OK) return rc;
    dw = dbias = nullptr;
  }
  const Pieces p = cut(n, channels, classes, dtype, dx, dw, dbias);
  if (p.bytes > workspace_bytes) return WCN_ERR_SCRATCH_TOO_SMALL;
  cudaStream_t st = wcn_stream(stream);
  char* const ws = (char*)workspace;
  const int e = wcn_dtype_size(dtype);
  const float lift = lift_of(dtype);
  wcn_ce_scale scale = {row_max ? row_max : grad, count, dtype == WCN_F16 ? 1.f / 16384.f : 1.f, late ? grad : nullptr, labels, ignore, classes};
  if (p.head) {
    wcn_ce_piece q = {};
    q.x = x; q.w = w; q.x_ld = x_ld; q.w_ld = w_ld; q.rows = (int)n; q.classes = (int)classes; q.channels = channels; q.bias2 = bias2;
    q.lse2 = lse2; q.loss = loss_rows; q.labels = labels; q.ignore = ignore; q.all_classes = classes;
    q.row_scale = row_max && !late ? grad : nullptr; q.row_max = row_max;
    float *const slab = dw || dbias ? (float*)(ws + p.slab_w) : nullptr, *const ones = dbias ? (float*)(ws + p.slab_b) : nullptr;
    int rc = wcn_ce_head(q, scale, dx, slab, ones, dtype, lift, dev_status, st);
    const JoinParams for_w = {slab, nullptr, false, dw, classes, channels, p.ld, p.head, scale, dev_status}, for_b = {ones, nullptr, false, dbias, classes, 1, 1, p.head, scale, dev_status};
    if (rc == WCN_OK && dw && dbias && bias_dtype == dtype) return join_both(for_w, for_b, dtype, st);
    if (rc == WCN_OK && dw) rc = join(for_w, dtype, st);
    if (rc == WCN_OK && dbias) rc = join(for_b, bias_dtype, st);
    return rc;
  }
  for (int i = 0; i < p.row_pieces; ++i) {
    const int64_t r0 = (int64_t)i * p.rows;
    const int rows = (int)(n - r0 < p.rows ? n - r0 : p.rows);
    for (int j = 0; j < p.class_pieces; ++j) {
      const int64_t v0 = (int64_t)j * p.classes;
      const int vs = (int)(classes - v0 < p.classes ? classes - v0 : p.classes);
      wcn_ce_piece q = {};
      q.x = (const char*)x + r0 * x_ld * e; q.w = (const char*)w + v0 * w_ld * e; q.x_ld = x_ld; q.w_ld = w_ld;
      q.rows = rows; q.classes = vs; q.channels = channels; q.bias2 = bias2 ? bias2 + v0 : nullptr;
      q.lse2 = lse2 + r0; q.loss = loss_rows + r0; q.labels = labels + r0; q.ignore = ignore; q.first_class = v0; q.all_classes = classes;
      q.row_scale = row_max && !late ? grad + r0 : nullptr; q.row_max = row_max;
      if (late) { scale.rows = grad + r0; scale.labels = labels + r0; }
      q.g = ws + p.g; q.g_ld = p.g_ld;
      int rc = WCN_OK;
      if (p.fused) {
        int chunk, slots;
        wcn_ce_rows_plan(rows, vs, &chunk, &slots);
        if (!dw && !dbias) q.g = nullptr;
        float* const slab = dx ? (float*)(ws + p.slab_x) : nullptr;
        rc = wcn_ce_rows(q, slab, dtype, lift, dev_status, st);
        if (rc == WCN_OK && dx)
          rc = join({slab, (float*)(ws + p.acc_x), j > 0, j == p.class_pieces - 1 ? (char*)dx + r0 * channels * e : nullptr, rows, channels, p.ld, slots, scale, dev_status,
                     (vs + 127) / 128, chunk}, dtype, st);
      } else if (dtype == WCN_F32) {
        ce_logits_fp32_kernel<true><<<dim3((rows + TILE - 1) / TILE, (vs + TILE - 1) / TILE), THREADS, 0, st>>>(q, 1);
        ++wcn_launched;
      } else rc = wcn_ce_logits(q, nullptr, dtype, true, lift, dev_status, st);
      if (rc != WCN_OK) return rc;
      if (dx && !p.fused) {
        wcn_ce_product d = {};
        d.a = q.g; d.a_ld = p.g_ld; d.b = q.w; d.b_ld = w_ld; d.m = rows; d.n = channels; d.k = vs;
        d.splits = product_splits(rows, channels, vs, dtype); d.slab = (float*)(ws + p.slab_x); d.scale = scale;
        char* const out = (char*)dx + r0 * channels * e;
        const bool whole = p.class_pieces == 1 && d.splits == 1 && dtype != WCN_F32;
        if (whole) d.out = out;
        rc = dtype == WCN_F32 ? fp32_product(d, false, st) : wcn_ce_product_run(d, false, false, dtype, dev_status, st);
        if (rc != WCN_OK) return rc;
        if (!whole) {
          JoinParams jp = {d.slab, (float*)(ws + p.acc_x), j > 0, j == p.class_pieces - 1 ? out : nullptr, rows, channels, p.ld, d.splits, scale, dev_status};
          rc = join(jp, dtype, st);
          if (rc != WCN_OK) return rc;
        }
      }
      if (dw || dbias) {
        wcn_ce_product d = {};
        d.a = q.g; d.a_ld = p.fused ? (vs + 127) / 128 : p.g_ld; d.b = q.x; d.b_ld = x_ld; d.m = vs; d.n = channels; d.k = rows;
        d.splits = product_splits(vs, channels, rows, dtype, p.fused, dbias); d.slab = (float*)(ws + p.slab_w); d.scale = scale;
        d.slab_ones = dbias ? (float*)(ws + p.slab_b) : nullptr;
        rc = dtype == WCN_F32 ? fp32_product(d, true, st) : wcn_ce_product_run(d, true, p.fused, dtype, dev_status, st);
        if (rc != WCN_OK) return rc;
        const bool done = i == p.row_pieces - 1;
        if (dw && dbias && p.row_pieces == 1 && dtype == bias_dtype && d.splits >= 16) {
          rc = join_both({d.slab, nullptr, false, (char*)dw + v0 * channels * e, vs, channels, p.ld, d.splits, scale, dev_status},
                         {d.slab_ones, nullptr, false, (char*)dbias + v0 * e, vs, 1, 1, d.splits, scale, dev_status}, dtype, st);
          if (rc != WCN_OK) return rc;
          continue;
        }
        if (dw) {
          JoinParams jp = {d.slab, (float*)(ws + p.acc_w) + v0 * p.ld, i > 0, done ? (char*)dw + v0 * channels * e : nullptr, vs, channels, p.ld, d.splits, scale, dev_status};
          rc = join(jp, dtype, st);
          if (rc != WCN_OK) return rc;
        }
        if (dbias) {
          JoinParams jp = {d.slab_ones, (float*)(ws + p.acc_b) + v0, i > 0, done ? (char*)dbias + v0 * wcn_dtype_size(bias_dtype) : nullptr, vs, 1, 1, d.splits, scale, dev_status};
          rc = join(jp, bias_dtype, st);
          if (rc != WCN_OK) return rc;
        }
      }
    }
  }
  return cudaGetLastError() == cudaSuccess ? WCN_OK : WCN_ERR_EXECUTION;
}
