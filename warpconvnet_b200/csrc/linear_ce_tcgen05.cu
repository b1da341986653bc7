// The matrix products of the linear cross entropy in 16 bits on the tensor cores.
//
// ce_logits_kernel computes tiles of 128 rows x up to 256 classes of z = x w^T + b and uses them as they leave tensor memory:
//   forward   running (largest, sum of exponentials) of each row over the classes of a unit, one pair per quarter of a tile's columns;
//   backward  g = (softmax - onehot) in 16 bits, a piece of the gradient of the logits, from the saved log-sum-exp.
// ce_product_kernel multiplies such a piece by the weights (dX = g W) or by the rows (dW = g^T X).
//
// Logits are kept in units of ln 2, so that an exponential is one instruction.  Both kernels are persistent: one thread issues
// TMA tile loads into a ring, one the matrix instructions, eight or sixteen warps empty one of two accumulators while the other is filled.
// Where they fit, the rows of a tile (up to 384 channels) or the classes (up to 256 of them) stay in shared memory and only the
// other operand passes: a multiprocessor receives about 80 bytes a clock, and a tile whose operands both arrived anew would
// wait for them (192 KB against 2 048 clocks of matrix instructions at 256 channels).
//
// Measured: logits and sums of 30 000 rows x 256 channels x 32 768 classes bf16 in 388 to 436 us, 1.2 to 1.3 PFLOP/s, where matrix
// instructions and the power cap bound them; of 60 000 x 128 x 4 096 fp16 in 94 us, 0.67 PFLOP/s, where the exponentials do (the
// special-function pipe is 73 % busy, the tensor pipe 35 %; a quarter of them as polynomials on the FMA pipe gained 2 %, more lost;
// the label's logit, row by row or by a comparison of each number, 6 to 8 %: see ce_loss_kernel for how it is had).  dw of 15 000 x
// 256 x 16 384 in 105 to 113 us, 1.1 to 1.2 PFLOP/s; with half as many splits, from an estimate by narrower tiles than it had, it
// took 178.
//
// Every wait is bounded (tcgen05_common.cuh); a kernel that gives up sets the status word, waits for its copies and matrix
// instructions and frees its tensor memory; what was to come of it is then filled with NaN (linear_ce.cu).
#include "linear_ce.cuh"
#include "tcgen05_common.cuh"
#include "tma_common.cuh"

namespace {

constexpr int TILE_M = 128, SLICE = 64;                   // rows of a tile; channels (elements of k) of a stage
constexpr int A_BYTES = TILE_M * SLICE * 2;
constexpr int MAX_STAGES = 12;
constexpr int EPI_WARP0 = 2;
constexpr int PARTS = 4, LOGIT_WARPS = 4 * PARTS, LOGIT_THREADS = (EPI_WARP0 + LOGIT_WARPS) * 32;   // four warps a lane quarter share a tile's columns
constexpr int EPI_WARPS = 8, THREADS = (EPI_WARP0 + EPI_WARPS) * 32;
constexpr int SMEM_BUDGET = 222 * 1024;
constexpr float LOG2E = 1.4426950408889634f;

struct Ring {
  int slot, phase, depth;
  __device__ __forceinline__ void advance() {
    if (++slot == depth) { slot = 0; phase ^= 1; }
  }
};

struct Control {
  uint64_t full[MAX_STAGES], empty[MAX_STAGES];
  uint64_t res_full, res_empty;
  uint64_t acc_full[2], acc_empty[2];
  uint64_t done;
  uint32_t tmem_holder;
  int32_t skip;
};

__device__ __forceinline__ uint32_t bar(uint64_t* b) { return smem_u32(b); }

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, "
      "%20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&r)[32]) { tmem_ld32(taddr, r); }
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&r)[16]) { tmem_ld16(taddr, r); }

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <bool BF16> __device__ __forceinline__ uint32_t pack2(float a, float b) {
  if (BF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Barriers, tensor memory and the look at the status word that both kernels begin with; false: an earlier launch gave up.
__device__ __forceinline__ bool begin(Control* ctl, int stages, int tmem_cols, int epi_warps, int32_t* dev_status) {
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) ctl->skip = *(volatile int32_t*)dev_status;
  __syncthreads();
  if (ctl->skip == (int)WCN_ERR_WAIT_EXPIRED) return false;
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) { mbar_init(bar(&ctl->full[s]), 1); mbar_init(bar(&ctl->empty[s]), 1); }
    mbar_init(bar(&ctl->res_full), 1);
    mbar_init(bar(&ctl->res_empty), 1);
    for (int i = 0; i < 2; ++i) { mbar_init(bar(&ctl->acc_full[i]), 1); mbar_init(bar(&ctl->acc_empty[i]), (uint32_t)epi_warps); }
    mbar_init(bar(&ctl->done), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc(smem_u32(&ctl->tmem_holder), (uint32_t)tmem_cols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  return true;
}

// A producer that gave up: the copies it has issued land before the block's shared memory is given back.  (The ring stands
// behind the last fill; fill i of a slot completes phase i & 1 of its barrier.)
__device__ void drain_ring(Control* ctl, Ring r, int issued) {
  for (int i = 0; i < issued && i < r.depth; ++i) {
    if (--r.slot < 0) { r.slot = r.depth - 1; r.phase ^= 1; }
    for (int k = 0; k < 100000 && !mbar_try_wait(bar(&ctl->full[r.slot]), (uint32_t)r.phase); ++k) {}
  }
}

// ------------------------------------------------------------------ logits

enum Resident { NOTHING = 0, ROWS = 1, CLASSES = 2 };

struct LogitParams {
  wcn_ce_piece q;
  wcn_ce_result out;      // forward with the classes resident
  int KB;                 // slices of 64 channels
  int NT;                 // classes of a tile
  int m_tiles, n_tiles, splits, per, units, stages, tmem_cols;
  float lift;             // exponent that gradients are raised by (fp16: 14)
  int32_t* dev_status;
};

// Logits in units of ln 2 from W accumulators, columns `col` on; -inf behind the last class.
template <int W> __device__ __forceinline__ void to_logits(const wcn_ce_piece& q, const uint32_t (&r)[W], int col, float (&z)[W]) {
  if (q.bias2) {
#pragma unroll
    for (int i = 0; i < W; i += 4) {
      const float4 b = *reinterpret_cast<const float4*>(q.bias2 + col + i);
      z[i] = fmaf(__uint_as_float(r[i]), LOG2E, b.x);
      z[i + 1] = fmaf(__uint_as_float(r[i + 1]), LOG2E, b.y);
      z[i + 2] = fmaf(__uint_as_float(r[i + 2]), LOG2E, b.z);
      z[i + 3] = fmaf(__uint_as_float(r[i + 3]), LOG2E, b.w);
    }
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i) z[i] = __uint_as_float(r[i]) * LOG2E;
    if (col + W > q.classes) {
#pragma unroll
      for (int i = 0; i < W; ++i)
        if (col + i >= q.classes) z[i] = -INFINITY;
    }
  }
}

// What the gradient of a row's logits needs: the exponent's shift (-inf: the row does not count), the gradient of its loss, its
// label's column of the piece (-1: elsewhere) and the gradient there.
struct RowGrad {
  float minus, scale;
  int label;
};
__device__ __forceinline__ RowGrad row_grad(const wcn_ce_piece& q, int row, float lift) {
  RowGrad g = {-INFINITY, 1.f, -1};
  if (row >= q.rows) return g;
  const int64_t y = __ldg(&q.labels[row]);
  if (y == q.ignore || y < 0 || y >= q.all_classes) return g;
  g.minus = lift - __ldg(&q.lse2[row]);
  const int64_t in = y - q.first_class;
  g.label = in >= 0 && in < q.classes ? (int)in : -1;
  if (q.row_scale) {
    const float most = __ldg(q.row_max);
    g.scale = __ldg(&q.row_scale[row]) / (most > 0.f ? most : 1.f);
  }
  return g;
}
// softmax - 1 at the label's class, from the row's loss: no difference of nearly equal numbers.
template <bool BF16> __device__ __forceinline__ uint16_t label_grad(const wcn_ce_piece& q, const RowGrad& g, int row, float lift) {
  const float d = expm1f(-__ldg(&q.loss[row])) * g.scale * exp2f(lift);
  return (uint16_t)pack2<BF16>(d, d);
}
template <int W, bool BF16> __device__ __forceinline__ void gradients(const wcn_ce_piece& q, const RowGrad& g, const float (&z)[W], uint32_t (&out)[W / 2]) {
#pragma unroll
  for (int i = 0; i < W; i += 2) {
    float a = exp2_fast(z[i] + g.minus), b = exp2_fast(z[i + 1] + g.minus);
    if (q.row_scale) { a *= g.scale; b *= g.scale; }
    out[i / 2] = g.minus == -INFINITY ? 0u : pack2<BF16>(a, b);   // (a row that does not count, whatever is in it)
  }
}

// What the parts of a row come to together, in shared memory (forward with the classes resident: a tile has whole rows).
struct WholeRows {
  float bias2[256];
  float4 part[2][PARTS][TILE_M];      // (largest, sum, the label's logit if it is this part's); tiles in turns
  uint64_t full[2], empty[2];
  double sums[4];
  int counts[4];
  int last;
};

__device__ __forceinline__ float bias_at(const wcn_ce_result& o, int i) {
  if (o.bias_dtype == WCN_F32) return reinterpret_cast<const float*>(o.bias)[i];
  if (o.bias_dtype == WCN_F16) return __half2float(reinterpret_cast<const __half*>(o.bias)[i]);
  return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(o.bias)[i]);
}

// The block's sum of losses, and of the last block to get here the mean or the sum (in a fixed order).
__device__ void finish_loss(const wcn_ce_result& o, WholeRows* w, bool failed) {
  if (threadIdx.x == 0) {
    double total = 0;
    int counted = 0;
    for (int i = 0; i < 4; ++i) { total += w->sums[i]; counted += w->counts[i]; }
    o.block_sums[blockIdx.x] = failed ? (double)__int_as_float(0x7FC00000) : total;
    o.block_counts[blockIdx.x] = counted;
    __threadfence();
    w->last = atomicAdd(o.counter, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (!w->last || threadIdx.x >= 32) return;
  __threadfence();
  double total = 0;
  int counted = 0;
  for (int i = threadIdx.x; i < (int)gridDim.x; i += 32) {
    total += __ldcg(&o.block_sums[i]);
    counted += __ldcg(&o.block_counts[i]);
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    total += __shfl_xor_sync(0xFFFFFFFFu, total, d);
    counted += __shfl_xor_sync(0xFFFFFFFFu, counted, d);
  }
  if (threadIdx.x == 0) {
    *o.loss = (float)(o.reduction == 1 ? total / (double)counted : total);
    *o.count = counted;
    *o.counter = 0;
  }
}

template <int RES, bool GRAD, bool BF16>
__global__ void __launch_bounds__(LOGIT_THREADS, 1)
ce_logits_kernel(const __grid_constant__ CUtensorMap x_map, const __grid_constant__ CUtensorMap w_map, const __grid_constant__ LogitParams p) {
  extern __shared__ uint8_t smem_raw[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int B_BYTES = p.NT * SLICE * 2;
  const int stage_bytes = RES == ROWS ? B_BYTES : RES == CLASSES ? A_BYTES : A_BYTES + B_BYTES;
  const int res_slice = RES == ROWS ? A_BYTES : B_BYTES;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t res = base + (uint32_t)(p.stages * stage_bytes);
  Control* ctl = reinterpret_cast<Control*>(smem_raw + (base - smem_u32(smem_raw)) + p.stages * stage_bytes + (RES == NOTHING ? 0 : p.KB * res_slice));
  constexpr bool WHOLE = RES == CLASSES && !GRAD;           // losses are finished here
  WholeRows* const whole = reinterpret_cast<WholeRows*>(reinterpret_cast<uint8_t*>(ctl) + (sizeof(Control) + 15) / 16 * 16);
  auto mark = [&]() {   // no losses of this block's rows
    for (int u = blockIdx.x; u < p.units; u += gridDim.x)
      for (int r = threadIdx.x; r < TILE_M; r += LOGIT_THREADS)
        if (u * TILE_M + r < p.q.rows) p.out.lse2[u * TILE_M + r] = p.out.loss_rows[u * TILE_M + r] = __int_as_float(0x7FC00000);
  };
  wcn_ce_piece q = p.q;
  if (WHOLE) {
    if (threadIdx.x < 4) { whole->sums[threadIdx.x] = 0; whole->counts[threadIdx.x] = 0; }
    if (threadIdx.x == 0)
      for (int i = 0; i < 2; ++i) { mbar_init(bar(&whole->full[i]), LOGIT_WARPS); mbar_init(bar(&whole->empty[i]), 4); }
    if (p.out.bias) {
      for (int i = threadIdx.x; i < 256; i += LOGIT_THREADS) whole->bias2[i] = i < q.classes ? bias_at(p.out, i) * LOG2E : -INFINITY;
      if (blockIdx.x == 0)
        for (int i = threadIdx.x; i < 512; i += LOGIT_THREADS) p.out.bias2[i] = i < q.classes ? bias_at(p.out, i) * LOG2E : -INFINITY;
      q.bias2 = whole->bias2;
    }
  }
  if (!begin(ctl, p.stages, p.tmem_cols, LOGIT_WARPS, p.dev_status)) {
    if (WHOLE) {
      mark();
      __syncthreads();
      if (p.out.loss) finish_loss(p.out, whole, true);
    }
    return;
  }
  const uint32_t tmem = ctl->tmem_holder;
  bool ok = true;

  if (warp == 0) {
    if (elect_one()) {
      Ring r{0, 0, p.stages};
      int issued = 0, res_phase = 0;
      bool have = false;
      for (int u = blockIdx.x; u < p.units && ok; u += gridDim.x) {
        const int m = u % p.m_tiles, n0 = u / p.m_tiles * p.per, n1 = min(n0 + p.per, p.n_tiles);
        if (RES == ROWS || (RES == CLASSES && !have)) {
          if (!mbar_wait(bar(&ctl->res_empty), res_phase ^ 1, p.dev_status)) { ok = false; break; }
          res_phase ^= 1;
          have = true;
          const uint32_t full = bar(&ctl->res_full);
          mbar_expect_tx(full, (uint32_t)(p.KB * res_slice));
          for (int s = 0; s < p.KB; ++s)
            tma_load_2d(res + (uint32_t)(s * res_slice), RES == ROWS ? &x_map : &w_map, s * SLICE, RES == ROWS ? m * TILE_M : 0, full);
        }
        for (int n = n0; n < n1 && ok; ++n)
          for (int s = 0; s < p.KB; ++s) {
            if (!mbar_wait(bar(&ctl->empty[r.slot]), r.phase ^ 1, p.dev_status)) { ok = false; break; }
            const uint32_t full = bar(&ctl->full[r.slot]), at = base + (uint32_t)(r.slot * stage_bytes);
            mbar_expect_tx(full, (uint32_t)stage_bytes);
            if (RES != ROWS) tma_load_2d(at, &x_map, s * SLICE, m * TILE_M, full);
            if (RES != CLASSES) tma_load_2d(RES == NOTHING ? at + A_BYTES : at, &w_map, s * SLICE, n * p.NT, full);
            r.advance();
            ++issued;
          }
      }
      if (!ok) {
        drain_ring(ctl, r, issued);
        for (int k = 0; have && k < 100000 && !mbar_try_wait(bar(&ctl->res_full), (uint32_t)(res_phase ^ 1)); ++k) {}
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect_one()) {
      const uint32_t idesc = (1u << 4) | ((BF16 ? 1u : 0u) << 7) | ((BF16 ? 1u : 0u) << 10) | ((uint32_t)(p.NT >> 3) << 17) |
                             ((uint32_t)(TILE_M >> 4) << 24);
      Ring r{0, 0, p.stages};
      int ab = 0, aphase = 0, res_phase = 0;
      bool have = false;
      const uint64_t ring0 = smem_desc<128>(base), res0 = smem_desc<128>(res);
      for (int u = blockIdx.x; u < p.units && ok; u += gridDim.x) {
        const int n0 = u / p.m_tiles * p.per, n1 = min(n0 + p.per, p.n_tiles);
        if (RES == ROWS || (RES == CLASSES && !have)) {
          if (!mbar_wait(bar(&ctl->res_full), res_phase, p.dev_status)) { ok = false; break; }
          res_phase ^= 1;
          have = true;
        }
        for (int n = n0; n < n1 && ok; ++n) {
          if (!mbar_wait(bar(&ctl->acc_empty[ab]), aphase ^ 1, p.dev_status)) { ok = false; break; }
          tc_fence_after();
          const uint32_t d = tmem + (uint32_t)(ab * p.NT);
          for (int s = 0; s < p.KB; ++s) {
            if (!mbar_wait(bar(&ctl->full[r.slot]), r.phase, p.dev_status)) { ok = false; break; }
            tc_fence_after();
            const uint64_t ring = ring0 + (uint64_t)((r.slot * stage_bytes) >> 4), kept = res0 + (uint64_t)((s * res_slice) >> 4);
            const uint64_t a = RES == ROWS ? kept : ring, b = RES == CLASSES ? kept : RES == NOTHING ? ring + (A_BYTES >> 4) : ring;
#pragma unroll
            for (int k = 0; k < SLICE / 16; ++k) umma_f16(d, a + (uint64_t)(k * 2), b + (uint64_t)(k * 2), idesc, (s | k) ? 1u : 0u);
            umma_commit(bar(&ctl->empty[r.slot]));
            r.advance();
          }
          if (!ok) break;
          umma_commit(bar(&ctl->acc_full[ab]));
          if (++ab == 2) { ab = 0; aphase ^= 1; }
        }
        if (RES == ROWS) umma_commit(bar(&ctl->res_empty));
      }
      umma_commit(bar(&ctl->done));
      (void)mbar_wait(bar(&ctl->done), 0, p.dev_status);
    }
    __syncwarp();
  } else {
    const int quarter = warp & 3, part = (warp - EPI_WARP0) >> 2;
    const int pieces = p.NT / 16, first = pieces * part / PARTS, last = pieces * (part + 1) / PARTS;   // of 16 columns
    int ab = 0, aphase = 0, tiles = 0, counted = 0;
    double total = 0;
    bool bad = false;
    for (int u = blockIdx.x; u < p.units; u += gridDim.x) {
      const int m = u % p.m_tiles, split = u / p.m_tiles, n0 = split * p.per, n1 = min(n0 + p.per, p.n_tiles);
      const int row = m * TILE_M + quarter * 32 + lane;
      const bool live = row < p.q.rows;
      float top = -INFINITY, sum = 0.f;                  // forward
      RowGrad rg = {};                                   // backward
      if (GRAD) rg = row_grad(p.q, row, p.lift);
      const int64_t y = WHOLE && live ? __ldg(&p.q.labels[row]) : p.q.ignore;
      const bool counts = WHOLE && y != p.q.ignore && y >= 0 && y < p.q.all_classes;
      const int label = counts ? (int)y : -1;
      float z_label = -INFINITY;
      for (int n = n0; n < n1; ++n) {
        if (ok) ok = mbar_wait(bar(&ctl->acc_full[ab]), aphase, p.dev_status);
        if (!__all_sync(0xFFFFFFFFu, ok)) { ok = false; break; }
        tc_fence_after();
        const uint32_t t = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(ab * p.NT);
        const int col0 = n * p.NT;
        auto use = [&](auto& r, int c) {   // columns c .. of the tile
          constexpr int W = sizeof(r) / 4;
          __syncwarp();
          tmem_load(t + (uint32_t)c, r);
          tmem_ld_wait();
          float z[W];
          const int col = col0 + c;
          to_logits<W>(q, r, col, z);
          if (!GRAD) {
            float m8[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) m8[i] = z[i];
#pragma unroll
            for (int i = 8; i < W; ++i) m8[i & 7] = fmaxf(m8[i & 7], z[i]);
#pragma unroll
            for (int o = 4; o; o >>= 1)
#pragma unroll
              for (int i = 0; i < o; ++i) m8[i] = fmaxf(m8[i], m8[i + o]);
            const float now = fmaxf(top, m8[0]), by = now == -INFINITY ? 0.f : now;   // (a row of -inf so far: sums of zeros)
            float s4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < W; ++i) s4[i & 3] += exp2_fast(z[i] - by);
            sum = fmaf(sum, exp2_fast(top - by), (s4[0] + s4[1]) + (s4[2] + s4[3]));
            top = now;
            if (WHOLE) {
#pragma unroll
              for (int i = 0; i < W; ++i) z_label = col + i == label ? z[i] : z_label;
            }
          } else {
            uint32_t out[W / 2];
            gradients<W, BF16>(p.q, rg, z, out);
            uint16_t* const g = reinterpret_cast<uint16_t*>(p.q.g) + (int64_t)row * p.q.g_ld + col;
#pragma unroll
            for (int i = 0; i < W / 16; ++i)
              if (live && col + 16 * i < p.q.g_ld) st_global_32B(g + 16 * i, out + 8 * i);
            const int in = rg.label - col;
            if (in >= 0 && in < W) g[in] = label_grad<BF16>(p.q, rg, row, p.lift);
          }
        };
        int c = first;
        for (; c + 2 <= last; c += 2) { uint32_t r[32]; use(r, c * 16); }
        if (c < last) { uint32_t r[16]; use(r, c * 16); }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(&ctl->acc_empty[ab]));
        if (++ab == 2) { ab = 0; aphase ^= 1; }
      }
      if (!ok) break;
      if (WHOLE) {
        const int turn = tiles & 1, phase = (tiles >> 1) & 1;
        if (tiles > 1) ok = mbar_wait(bar(&whole->empty[turn]), phase ^ 1, p.dev_status);
        if (!__all_sync(0xFFFFFFFFu, ok)) { ok = false; break; }
        whole->part[turn][part][quarter * 32 + lane] = make_float4(top, sum, z_label, label >= 0 && label / 16 >= first && label / 16 < last ? 1.f : 0.f);
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(&whole->full[turn]));
        if (part == 0) {
          ok = mbar_wait(bar(&whole->full[turn]), phase, p.dev_status);
          if (!__all_sync(0xFFFFFFFFu, ok)) { ok = false; break; }
        }
        if (part == 0 && live) {
          float all = -INFINITY, s = 0.f, z = -INFINITY;
#pragma unroll
          for (int k = 0; k < PARTS; ++k) all = fmaxf(all, whole->part[turn][k][quarter * 32 + lane].x);
          const float by = all == -INFINITY ? 0.f : all;
#pragma unroll
          for (int k = 0; k < PARTS; ++k) {
            const float4 v = whole->part[turn][k][quarter * 32 + lane];
            s += v.y * exp2f(v.x - by);
            if (v.w != 0.f) z = v.z;
          }
          const float more = log2f(s);
          float loss = 0.f;
          if (counts) {
            loss = ((all - z) + more) * 0.69314718055994531f;
            if (loss < 0.f) loss = 0.f;                    // (roundings of a probability of one)
          }
          bad |= y != p.q.ignore && !counts;
          p.out.lse2[row] = all + more;
          p.out.loss_rows[row] = loss;
          total += (double)loss;
          counted += counts;
        }
        __syncwarp();
        if (part == 0 && lane == 0) mbar_arrive(bar(&whole->empty[turn]));
        ++tiles;
      } else if (!GRAD && live) {
        p.q.part[(int64_t)(split * PARTS + part) * p.q.rows + row] = make_float2(top, sum);
      }
    }
    if (WHOLE && part == 0) {
      if (bad) wcn_report_bounds(p.dev_status);
      __syncwarp();
#pragma unroll
      for (int o = 16; o; o >>= 1) {
        total += __shfl_xor_sync(0xFFFFFFFFu, total, o);
        counted += __shfl_xor_sync(0xFFFFFFFFu, counted, o);
      }
      if (lane == 0) { whole->sums[quarter] = total; whole->counts[quarter] = counted; }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, (uint32_t)p.tmem_cols);
  if (WHOLE) {
    if (threadIdx.x == 0) ctl->skip = *(volatile int32_t*)p.dev_status;
    __syncthreads();
    const bool failed = ctl->skip == (int)WCN_ERR_WAIT_EXPIRED;
    if (failed) mark();
    if (p.out.loss) finish_loss(p.out, whole, failed);
  }
}

// ------------------------------------------------------------------ products

struct ProductParams {
  wcn_ce_product q;
  int NT, NB;             // columns of a tile, chunks of 64 of them
  int m_tiles, n_tiles, units, ksteps, per, stages, accs, stride, tmem_cols;
  int vec;                // rows of `out` start on 32-byte boundaries
  int32_t* dev_status;
};

// BLOCKED: A is g as ce_rows_kernel leaves it, images of [128 rows][64 classes] with which a stage is filled as it is, for 256
// classes at a time: what arrives in shared memory is then 64 bytes a clock of the matrix instructions, with 128 classes 96.
template <bool TRANS, bool BLOCKED, bool BF16>
__global__ void __launch_bounds__(THREADS, 1)
ce_product_kernel(const __grid_constant__ CUtensorMap a_map, const __grid_constant__ CUtensorMap b_map, const __grid_constant__ ProductParams p) {
  extern __shared__ uint8_t smem_raw[];
  constexpr int CHUNK = SLICE * 128;                      // 64 rows of k x 64 columns
  constexpr int MB = BLOCKED ? 2 : 1;                     // blocks of 128 rows of a tile
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int stage_bytes = MB * A_BYTES + p.NB * CHUNK;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t ones = base + (uint32_t)(p.stages * stage_bytes);
  uint8_t* const gen = smem_raw + (base - smem_u32(smem_raw)) + p.stages * stage_bytes;
  Control* ctl = reinterpret_cast<Control*>(gen + CHUNK);
  const bool with_ones = p.q.slab_ones != nullptr;
  auto split_of = [&](int u) { return u / (p.m_tiles * p.n_tiles); };
  auto m_of = [&](int u) { return u / p.n_tiles % p.m_tiles; };
  auto n_of = [&](int u) { return u % p.n_tiles; };
  auto mark = [&]() {   // the finished result of this block's units, where it has none
    if (!p.q.out) return;
    const uint16_t nan = BF16 ? 0x7FC0 : 0x7E00;
    for (int u = blockIdx.x; u < p.units; u += gridDim.x)
      for (int i = threadIdx.x; i < MB * TILE_M * p.NT; i += THREADS) {
        const int row = m_of(u) * MB * TILE_M + i / p.NT, col = n_of(u) * p.NT + i % p.NT;
        if (row < p.q.m && col < p.q.n) reinterpret_cast<uint16_t*>(p.q.out)[(int64_t)row * p.q.n + col] = nan;
      }
  };
  if (with_ones) {   // a chunk of ones: the sums of A's rows are another 16 columns of the product
    const uint32_t one = BF16 ? 0x3F803F80u : 0x3C003C00u;
    for (int i = threadIdx.x; i < CHUNK / 4; i += THREADS) reinterpret_cast<uint32_t*>(gen)[i] = one;
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (!begin(ctl, p.stages, p.tmem_cols, EPI_WARPS, p.dev_status)) { mark(); return; }
  const uint32_t tmem = ctl->tmem_holder;
  bool ok = true;

  if (warp == 0) {
    if (elect_one()) {
      Ring r{0, 0, p.stages};
      int issued = 0;
      for (int u = blockIdx.x; u < p.units && ok; u += gridDim.x) {
        const int m = m_of(u) * MB * TILE_M, n = n_of(u) * p.NT, k0 = split_of(u) * p.per, k1 = min(k0 + p.per, p.ksteps);
        for (int k = k0; k < k1; ++k) {
          if (!mbar_wait(bar(&ctl->empty[r.slot]), r.phase ^ 1, p.dev_status)) { ok = false; break; }
          const uint32_t full = bar(&ctl->full[r.slot]), at = base + (uint32_t)(r.slot * stage_bytes);
          mbar_expect_tx(full, (uint32_t)stage_bytes);
          if (BLOCKED) {   // 64 rows of two images for each block of 128 classes (the last one again where there is no other)
#pragma unroll
            for (int j = 0; j < MB; ++j) {
              const int64_t tile = min((int64_t)(m / TILE_M + j), p.q.a_ld - 1);
              const char* const from = reinterpret_cast<const char*>(p.q.a) + ((int64_t)(k >> 1) * p.q.a_ld + tile) * (2 * A_BYTES) + (k & 1) * CHUNK;
              bulk_copy_g2s(at + j * A_BYTES, from, CHUNK, full);
              bulk_copy_g2s(at + j * A_BYTES + CHUNK, from + A_BYTES, CHUNK, full);
            }
          } else if (TRANS) {
            tma_load_2d(at, &a_map, m, k * SLICE, full);
            tma_load_2d(at + CHUNK, &a_map, m + 64, k * SLICE, full);
          } else {
            tma_load_2d(at, &a_map, k * SLICE, m, full);
          }
          for (int c = 0; c < p.NB; ++c) tma_load_2d(at + MB * A_BYTES + (uint32_t)(c * CHUNK), &b_map, n + 64 * c, k * SLICE, full);
          r.advance();
          ++issued;
        }
      }
      if (!ok) drain_ring(ctl, r, issued);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect_one()) {
      const uint32_t flags = (1u << 4) | ((BF16 ? 1u : 0u) << 7) | ((BF16 ? 1u : 0u) << 10) | (TRANS ? 1u << 15 : 0u) | (1u << 16) |
                             ((uint32_t)(TILE_M >> 4) << 24);
      const uint32_t idesc = flags | ((uint32_t)(p.NT >> 3) << 17), idesc_ones = flags | ((uint32_t)(16 >> 3) << 17);
      const uint64_t a0 = TRANS ? smem_desc_mn<128>(base, CHUNK) : smem_desc<128>(base), b0 = smem_desc_mn<128>(base + MB * A_BYTES, CHUNK);
      const uint64_t ones0 = smem_desc_mn<128>(ones, CHUNK);
      constexpr int A_STEP = TRANS ? 128 : 2;             // 16 of k further, in units of 16 bytes
      Ring r{0, 0, p.stages};
      int ab = 0, aphase = 0;
      for (int u = blockIdx.x; u < p.units && ok; u += gridDim.x) {
        const int k0 = split_of(u) * p.per, k1 = min(k0 + p.per, p.ksteps);
        const bool sums = with_ones && n_of(u) == 0;
        if (!mbar_wait(bar(&ctl->acc_empty[ab]), aphase ^ 1, p.dev_status)) { ok = false; break; }
        tc_fence_after();
        const uint32_t d0 = tmem + (uint32_t)(ab * MB * p.stride);
        for (int k = k0; k < k1; ++k) {
          if (!mbar_wait(bar(&ctl->full[r.slot]), r.phase, p.dev_status)) { ok = false; break; }
          tc_fence_after();
          const uint64_t at = (uint64_t)((r.slot * stage_bytes) >> 4);
#pragma unroll
          for (int j = 0; j < MB; ++j) {
            const uint64_t a = a0 + at + (uint64_t)((j * A_BYTES) >> 4);
            const uint32_t d = d0 + (uint32_t)(j * p.stride);
#pragma unroll
            for (int i = 0; i < SLICE / 16; ++i)
              umma_f16(d, a + (uint64_t)(i * A_STEP), b0 + at + (uint64_t)(i * 128), idesc, (k > k0 || i) ? 1u : 0u);
            if (sums)
#pragma unroll
              for (int i = 0; i < SLICE / 16; ++i)
                umma_f16(d + (uint32_t)p.NT, a + (uint64_t)(i * A_STEP), ones0 + (uint64_t)(i * 128), idesc_ones, (k > k0 || i) ? 1u : 0u);
          }
          umma_commit(bar(&ctl->empty[r.slot]));
          r.advance();
        }
        if (!ok) break;
        umma_commit(bar(&ctl->acc_full[ab]));
        if (++ab == p.accs) { ab = 0; aphase ^= 1; }
      }
      umma_commit(bar(&ctl->done));
      (void)mbar_wait(bar(&ctl->done), 0, p.dev_status);
    }
    __syncwarp();
  } else {
    const int quarter = warp & 3, half = (warp - EPI_WARP0) >> 2;
    const int pieces = p.NT / 16, first = half ? (pieces + 1) / 2 : 0, last = half ? pieces : (pieces + 1) / 2;
    const int64_t slab_ld = wcn_ce_round(p.q.n, 16);
    float scale = p.q.out && !p.q.scale.rows ? wcn_ce_factor(p.q.scale) : 0.f;
    int ab = 0, aphase = 0;
    for (int u = blockIdx.x; u < p.units; u += gridDim.x) {
      if (ok) ok = mbar_wait(bar(&ctl->acc_full[ab]), aphase, p.dev_status);
      if (!__all_sync(0xFFFFFFFFu, ok)) { ok = false; break; }
      tc_fence_after();
      const int n = n_of(u) * p.NT, split = split_of(u);
#pragma unroll 1
      for (int j = 0; j < MB; ++j) {
        const int row = (m_of(u) * MB + j) * TILE_M + quarter * 32 + lane;
        const bool live = row < p.q.m;
        if (p.q.out && p.q.scale.rows && live) scale = wcn_ce_row_factor(p.q.scale, row);
        const uint32_t t = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)((ab * MB + j) * p.stride);
        float* const slab = p.q.slab + ((int64_t)split * p.q.m + row) * slab_ld + n;
        uint16_t* const out = reinterpret_cast<uint16_t*>(p.q.out) + (int64_t)row * p.q.n + n;
        for (int c = first; c < last; ++c) {
          uint32_t r[16];
          __syncwarp();
          tmem_ld16(t + (uint32_t)(c * 16), r);
          tmem_ld_wait();
          if (!live) continue;
          if (p.q.out) {
            uint32_t v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = pack2<BF16>(__uint_as_float(r[2 * i]) * scale, __uint_as_float(r[2 * i + 1]) * scale);
            if (p.vec && n + c * 16 + 16 <= p.q.n) {
              st_global_32B(out + c * 16, v);
            } else {
#pragma unroll
              for (int i = 0; i < 16; ++i)
                if (n + c * 16 + i < p.q.n) out[c * 16 + i] = (uint16_t)(v[i / 2] >> (16 * (i & 1)));
            }
          } else if (n + c * 16 < slab_ld) {
            st_global_32B(slab + c * 16, r);
            st_global_32B(slab + c * 16 + 8, r + 8);
          }
        }
        if (with_ones && n == 0 && half) {
          uint32_t r[16];
          __syncwarp();
          tmem_ld16(t + (uint32_t)p.NT, r);
          tmem_ld_wait();
          if (live) p.q.slab_ones[(int64_t)split * p.q.m + row] = __uint_as_float(r[0]);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(&ctl->acc_empty[ab]));
      if (++ab == p.accs) { ab = 0; aphase ^= 1; }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, (uint32_t)p.tmem_cols);
  if (threadIdx.x == 0) ctl->skip = *(volatile int32_t*)p.dev_status;
  __syncthreads();
  if (ctl->skip == (int)WCN_ERR_WAIT_EXPIRED) mark();
}

// ------------------------------------------------------------------ gradients of few classes

// With at most 256 classes a tile's row of logits is whole, and both products can be made of g while it is in shared memory: x is
// read once, dx written once, and g is never in global memory.  Per 128 rows: z = x w^T; the epilogue warps write g as an operand
// tile; dx = g w and dw += g^T x, the latter in accumulators that stay in tensor memory until the block's last tile.  The same
// images in shared memory serve every product: a tile of rows whose channels (classes) run along 128-byte lines is a K-major
// operand with its rows on the M / N side, or an MN-major one with its rows on the K side.
// 240 000 x 96 x 200 classes bf16: 70 us, after 41 for the forward pass (reading and writing 92 MB would take 14); pieces of g
// through global memory took 64 (g) + 39 (dx) + 33 us (dw).  What bounds it is the chain of a tile, z -> g -> both products, of
// which tensor memory holds one set: 23 % of the tensor pipe and 59 MB of HBM traffic are used in that time.
struct HeadParams {
  wcn_ce_piece q;
  wcn_ce_scale scale;
  void* dx;               // [rows][channels] (null: not wanted)
  float* slab;            // [blocks][classes][channels rounded up to 16] (null: neither dw nor dbias)
  float* slab_ones;       // [blocks][classes] (null: no dbias)
  int KB, NT, CN, MB;     // slices of 64 channels; classes, channels rounded up to 16; blocks of 128 classes
  int apart;              // dx has columns of its own
  int acc, tmem_cols;     // first column of dw
  int tiles, vec;
  float lift;
  int32_t* dev_status;
};

struct HeadControl {
  uint64_t w_full, x_full[2], x_empty[2], s_full, g_full, g_empty, dx_full, dx_read, acc_full;
  uint32_t tmem_holder;
  int32_t skip;
};

constexpr int ONES_BYTES = 16 * 128;

template <bool BF16>
__global__ void __launch_bounds__(LOGIT_THREADS, 1)
ce_head_kernel(const __grid_constant__ CUtensorMap x_map, const __grid_constant__ CUtensorMap w_map, const __grid_constant__ HeadParams p) {
  extern __shared__ uint8_t smem_raw[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int w_slice = p.NT * 128, x_stage = p.KB * A_BYTES;
  const uint32_t pad = ((smem_u32(smem_raw) + 1023u) & ~1023u) - smem_u32(smem_raw);
  const int w_at = 0, x_at = w_at + p.KB * w_slice, g_at = x_at + 2 * x_stage, ones_at = g_at + p.MB * 2 * A_BYTES, ctl_at = ones_at + ONES_BYTES;
  uint8_t* const gen = smem_raw + pad;
  const uint32_t base = smem_u32(smem_raw) + pad;
  HeadControl* ctl = reinterpret_cast<HeadControl*>(gen + ctl_at);
  const bool sums = p.slab != nullptr, with_ones = p.slab_ones != nullptr;
  auto mark = [&]() {
    if (!p.dx) return;
    const uint16_t nan = BF16 ? 0x7FC0 : 0x7E00;
    for (int t = blockIdx.x; t < p.tiles; t += gridDim.x)
      for (int i = threadIdx.x; i < TILE_M * p.q.channels; i += LOGIT_THREADS) {
        const int row = t * TILE_M + i / p.q.channels;
        if (row < p.q.rows) reinterpret_cast<uint16_t*>(p.dx)[(int64_t)row * p.q.channels + i % p.q.channels] = nan;
      }
  };
  if (threadIdx.x == 0) ctl->skip = *(volatile int32_t*)p.dev_status;
  __syncthreads();
  if (ctl->skip == (int)WCN_ERR_WAIT_EXPIRED) { mark(); return; }
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) { mbar_init(bar(&ctl->x_full[i]), 1); mbar_init(bar(&ctl->x_empty[i]), 1); }
    mbar_init(bar(&ctl->w_full), 1);
    mbar_init(bar(&ctl->s_full), 1);
    mbar_init(bar(&ctl->g_full), LOGIT_WARPS);
    mbar_init(bar(&ctl->g_empty), 1);
    mbar_init(bar(&ctl->dx_full), 1);
    mbar_init(bar(&ctl->dx_read), LOGIT_WARPS);
    mbar_init(bar(&ctl->acc_full), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  const uint32_t one = BF16 ? 0x3F803F80u : 0x3C003C00u;
  for (int i = threadIdx.x; i < ONES_BYTES / 4; i += LOGIT_THREADS) reinterpret_cast<uint32_t*>(gen + ones_at)[i] = one;
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  if (warp == 1) tmem_alloc(smem_u32(&ctl->tmem_holder), (uint32_t)p.tmem_cols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctl->tmem_holder;
  const uint32_t dx_col = p.apart ? (uint32_t)p.NT : 0u;
  bool ok = true;

  if (warp == 0) {
    if (elect_one()) {
      mbar_expect_tx(bar(&ctl->w_full), (uint32_t)(p.KB * w_slice));
      for (int s = 0; s < p.KB; ++s) tma_load_2d(base + w_at + (uint32_t)(s * w_slice), &w_map, s * SLICE, 0, bar(&ctl->w_full));
      int i = 0;
      for (int t = blockIdx.x; t < p.tiles; t += gridDim.x, ++i) {
        if (!mbar_wait(bar(&ctl->x_empty[i & 1]), ((i >> 1) & 1) ^ 1, p.dev_status)) { ok = false; break; }
        const uint32_t full = bar(&ctl->x_full[i & 1]);
        mbar_expect_tx(full, (uint32_t)x_stage);
        for (int s = 0; s < p.KB; ++s) tma_load_2d(base + x_at + (uint32_t)((i & 1) * x_stage + s * A_BYTES), &x_map, s * SLICE, t * TILE_M, full);
      }
      if (!ok) {   // what has been issued lands before the block's shared memory is given back
        for (int k = 0; k < 100000 && !mbar_try_wait(bar(&ctl->w_full), 0); ++k) {}
        for (int j = i - 2 < 0 ? 0 : i - 2; j < i; ++j)
          for (int k = 0; k < 100000 && !mbar_try_wait(bar(&ctl->x_full[j & 1]), (uint32_t)((j >> 1) & 1)); ++k) {}
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect_one()) {
      const uint32_t flags = (1u << 4) | ((BF16 ? 1u : 0u) << 7) | ((BF16 ? 1u : 0u) << 10) | ((uint32_t)(TILE_M >> 4) << 24);
      const uint32_t n_s = (uint32_t)(p.NT >> 3) << 17, n_c = (uint32_t)(p.CN >> 3) << 17, n_one = 2u << 17;
      const uint32_t id_s = flags | n_s, id_dx = flags | (1u << 16) | n_c, id_dw = flags | (1u << 15) | (1u << 16) | n_c,
                     id_one = flags | (1u << 15) | (1u << 16) | n_one;
      const uint64_t w_k = smem_desc<128>(base + w_at), w_mn = smem_desc_mn<128>(base + w_at, (uint32_t)w_slice);
      const uint64_t x_k = smem_desc<128>(base + x_at), x_mn = smem_desc_mn<128>(base + x_at, A_BYTES);
      const uint64_t g_k = smem_desc<128>(base + g_at), g_mn = smem_desc_mn<128>(base + g_at, A_BYTES), ones = smem_desc_mn<128>(base + ones_at, ONES_BYTES);
      auto logits = [&](int i) {
        if (!mbar_wait(bar(&ctl->x_full[i & 1]), (i >> 1) & 1, p.dev_status)) { ok = false; return; }
        tc_fence_after();
        for (int s = 0; s < p.KB; ++s)
#pragma unroll
          for (int k = 0; k < SLICE / 16; ++k)
            umma_f16(tmem, x_k + (uint64_t)(((i & 1) * x_stage + s * A_BYTES) >> 4) + (uint64_t)(k * 2), w_k + (uint64_t)((s * w_slice) >> 4) + (uint64_t)(k * 2),
                     id_s, (s | k) ? 1u : 0u);
        umma_commit(bar(&ctl->s_full));
      };
      ok = mbar_wait(bar(&ctl->w_full), 0, p.dev_status);
      if (ok) logits(0);
      int i = 0;
      for (int t = blockIdx.x; t < p.tiles && ok; t += gridDim.x, ++i) {
        const bool more = t + (int)gridDim.x < p.tiles;
        if (!mbar_wait(bar(&ctl->g_full), i & 1, p.dev_status)) { ok = false; break; }
        tc_fence_after();
        if (p.dx) {
          for (int k = 0; k < p.NT / 16; ++k)   // 16 classes a step: a chunk of 64 is 16 KB of g and 64 lines of w
            umma_f16(tmem + dx_col, g_k + (uint64_t)(((k >> 2) * A_BYTES) >> 4) + (uint64_t)((k & 3) * 2), w_mn + (uint64_t)(k * 128), id_dx, k ? 1u : 0u);
          umma_commit(bar(&ctl->dx_full));
        }
        if (more && (p.apart || !p.dx)) {
          logits(i + 1);
          if (!ok) break;
        }
        if (sums) {
          const uint64_t x = x_mn + (uint64_t)(((i & 1) * x_stage) >> 4);
          for (int m = 0; m < p.MB; ++m) {
            const uint64_t g = g_mn + (uint64_t)((m * 2 * A_BYTES) >> 4);
            const uint32_t d = tmem + (uint32_t)(p.acc + m * p.CN);
#pragma unroll
            for (int k = 0; k < TILE_M / 16; ++k) umma_f16(d, g + (uint64_t)(k * 128), x + (uint64_t)(k * 128), id_dw, (i | k) ? 1u : 0u);
            if (with_ones) {
              const uint32_t d1 = tmem + (uint32_t)(p.acc + p.MB * p.CN + m * 16);
#pragma unroll
              for (int k = 0; k < TILE_M / 16; ++k) umma_f16(d1, g + (uint64_t)(k * 128), ones, id_one, (i | k) ? 1u : 0u);
            }
          }
        }
        umma_commit(bar(&ctl->x_empty[i & 1]));
        umma_commit(bar(&ctl->g_empty));
        if (more && !p.apart && p.dx) {
          if (!mbar_wait(bar(&ctl->dx_read), i & 1, p.dev_status)) { ok = false; break; }
          logits(i + 1);
        }
      }
      umma_commit(bar(&ctl->acc_full));
      (void)mbar_wait(bar(&ctl->acc_full), 0, p.dev_status);
    }
    __syncwarp();
  } else {
    const int quarter = warp & 3, part = (warp - EPI_WARP0) >> 2, in_tile = quarter * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
    const int pieces = p.NT / 16, first = pieces * part / PARTS, last = pieces * (part + 1) / PARTS;
    const int c_pieces = p.CN / 16, c_first = c_pieces * part / PARTS, c_last = c_pieces * (part + 1) / PARTS;
    float scale = p.dx && !p.scale.rows ? wcn_ce_factor(p.scale) : 0.f;
    int i = 0;
    RowGrad next = row_grad(p.q, (int)blockIdx.x * TILE_M + in_tile, p.lift);
    for (int t = blockIdx.x; t < p.tiles; t += gridDim.x, ++i) {
      const int row = t * TILE_M + in_tile;
      const RowGrad rg = next;
      next = row_grad(p.q, t + (int)gridDim.x < p.tiles ? row + (int)gridDim.x * TILE_M : p.q.rows, p.lift);
      if (ok) ok = mbar_wait(bar(&ctl->s_full), i & 1, p.dev_status);
      if (ok && i) ok = mbar_wait(bar(&ctl->g_empty), (i - 1) & 1, p.dev_status);
      if (!__all_sync(0xFFFFFFFFu, ok)) { ok = false; break; }
      tc_fence_after();
      for (int c = first; c < last; ++c) {
        uint32_t r[16], out[8];
        float z[16];
        __syncwarp();
        tmem_ld16(lanes + (uint32_t)(c * 16), r);
        tmem_ld_wait();
        to_logits<16>(p.q, r, c * 16, z);
        gradients<16, BF16>(p.q, rg, z, out);
        uint8_t* const chunk = gen + g_at + (c >> 2) * A_BYTES;
        const int piece = (c & 3) * 2;
        *reinterpret_cast<uint4*>(chunk + tile_offset<128>(in_tile, piece)) = make_uint4(out[0], out[1], out[2], out[3]);
        *reinterpret_cast<uint4*>(chunk + tile_offset<128>(in_tile, piece + 1)) = make_uint4(out[4], out[5], out[6], out[7]);
        const int in = rg.label - c * 16;
        if (in >= 0 && in < 16)
          reinterpret_cast<uint16_t*>(chunk + tile_offset<128>(in_tile, piece + (in >> 3)))[in & 7] = label_grad<BF16>(p.q, rg, row, p.lift);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(&ctl->g_full));
      if (!p.dx) continue;
      if (p.scale.rows && row < p.q.rows) scale = wcn_ce_row_factor(p.scale, row);
      if (ok) ok = mbar_wait(bar(&ctl->dx_full), i & 1, p.dev_status);
      if (!__all_sync(0xFFFFFFFFu, ok)) { ok = false; break; }
      tc_fence_after();
      uint16_t* const out = reinterpret_cast<uint16_t*>(p.dx) + (int64_t)row * p.q.channels;
      for (int c = c_first; c < c_last; ++c) {
        uint32_t r[16];
        __syncwarp();
        tmem_ld16(lanes + dx_col + (uint32_t)(c * 16), r);
        tmem_ld_wait();
        if (row >= p.q.rows) continue;
        uint32_t v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = pack2<BF16>(__uint_as_float(r[2 * k]) * scale, __uint_as_float(r[2 * k + 1]) * scale);
        if (p.vec && c * 16 + 16 <= p.q.channels) {
          st_global_32B(out + c * 16, v);
        } else {
#pragma unroll
          for (int k = 0; k < 16; ++k)
            if (c * 16 + k < p.q.channels) out[c * 16 + k] = (uint16_t)(v[k / 2] >> (16 * (k & 1)));
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(&ctl->dx_read));
    }
    if (sums) {
      __syncwarp();
      if (ok) ok = mbar_wait(bar(&ctl->acc_full), 0, p.dev_status);
      if (__all_sync(0xFFFFFFFFu, ok)) {
        tc_fence_after();
        for (int m = 0; m < p.MB; ++m) {
          const int cls = m * 128 + in_tile;
          const bool live = cls < p.q.classes;
          float* const to = p.slab + ((int64_t)blockIdx.x * p.q.classes + cls) * p.CN;
          for (int c = c_first; c < c_last; ++c) {
            uint32_t r[16];
            __syncwarp();
            tmem_ld16(lanes + (uint32_t)(p.acc + m * p.CN + c * 16), r);
            tmem_ld_wait();
            if (!live) continue;
            st_global_32B(to + c * 16, r);
            st_global_32B(to + c * 16 + 8, r + 8);
          }
          if (with_ones && part == PARTS - 1) {
            uint32_t r[16];
            __syncwarp();
            tmem_ld16(lanes + (uint32_t)(p.acc + p.MB * p.CN + m * 16), r);
            tmem_ld_wait();
            if (live) p.slab_ones[(int64_t)blockIdx.x * p.q.classes + cls] = __uint_as_float(r[0]);
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, (uint32_t)p.tmem_cols);
  if (threadIdx.x == 0) ctl->skip = *(volatile int32_t*)p.dev_status;
  __syncthreads();
  if (ctl->skip == (int)WCN_ERR_WAIT_EXPIRED) mark();
}

// ------------------------------------------------------------------ gradients of many classes

// g and dx = g w in one kernel, for up to 256 channels: the rows of a tile stay in shared memory, classes pass in tiles of 128;
// a tile's z = x w^T is computed in one of two accumulators while the epilogue warps turn the other into g, an operand tile in
// shared memory, of which dx += g w is made (in columns that stay in tensor memory for all classes of a row tile) and which one
// bulk copy leaves in global memory for dw, as it is: [128 rows][64 classes] images.  The (row tile, class tile) pairs are one
// sequence that is divided evenly among the blocks; where a row tile's classes are several blocks', each leaves its dx apart.
// As two kernels, the second of which read g again in rows of 128 bytes, 15 000 rows x 6 656 classes x 256 channels bf16 took
// 85 (g) + 62 us (dx); 15 000 x 16 384 x 256 takes 248 to 298, 0.85 to 1.0 PFLOP/s, with the tensor pipe 46 % busy: a tile's g has one
// place in shared memory, where the products of one tile and the exponentials of the next meet.  (g handed over in halves of 64
// classes, for more of the two at a time, made the whole call 2 % longer.)
struct RowsParams {
  wcn_ce_piece q;         // g: images, or null (no dw)
  float* slab;            // [slots][rows][channels rounded up to 16], or null (no dx)
  int KB, CN;
  int n_tiles, total, chunk;   // class tiles; pairs in all, and of a block
  float lift;
  int32_t* dev_status;
};

struct RowsControl {
  uint64_t x_full, x_empty, w_full[2], w_empty[2], s_full[2], g_full, g_empty, dx_full, dx_read, done;
  uint32_t tmem_holder;
  int32_t skip;
};

constexpr int STORE_WARP = 2, ROWS_WARP0 = 3, ROWS_THREADS = (ROWS_WARP0 + LOGIT_WARPS) * 32;
constexpr int ROWS_SMEM = 227 * 1024;

template <bool BF16>
__global__ void __launch_bounds__(ROWS_THREADS, 1)
ce_rows_kernel(const __grid_constant__ CUtensorMap x_map, const __grid_constant__ CUtensorMap w_map, const __grid_constant__ RowsParams p) {
  extern __shared__ uint8_t smem_raw[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slices = p.KB * A_BYTES;                       // a tile of 128 rows, or of 128 classes
  const uint32_t pad = ((smem_u32(smem_raw) + 1023u) & ~1023u) - smem_u32(smem_raw);
  const int x_at = 0, w_at = slices, g_at = 3 * slices;
  uint8_t* const gen = smem_raw + pad;
  const uint32_t base = smem_u32(smem_raw) + pad;
  RowsControl* ctl = reinterpret_cast<RowsControl*>(gen + g_at + 2 * A_BYTES);
  const bool want_x = p.slab != nullptr, want_w = p.q.g != nullptr;
  if (threadIdx.x == 0) ctl->skip = *(volatile int32_t*)p.dev_status;
  __syncthreads();
  if (ctl->skip == (int)WCN_ERR_WAIT_EXPIRED) return;
  if (threadIdx.x == 0) {
    mbar_init(bar(&ctl->x_full), 1);
    mbar_init(bar(&ctl->x_empty), 1);
    for (int i = 0; i < 2; ++i) { mbar_init(bar(&ctl->w_full[i]), 1); mbar_init(bar(&ctl->w_empty[i]), 1); mbar_init(bar(&ctl->s_full[i]), 1); }
    mbar_init(bar(&ctl->g_full), LOGIT_WARPS);
    mbar_init(bar(&ctl->g_empty), 2);                      // the products that read g, and the copy of it
    mbar_init(bar(&ctl->dx_full), 1);
    mbar_init(bar(&ctl->dx_read), LOGIT_WARPS);
    mbar_init(bar(&ctl->done), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc(smem_u32(&ctl->tmem_holder), 512u);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctl->tmem_holder, dx_col = 256;
  const int begin_at = (int)blockIdx.x * p.chunk, end_at = min(begin_at + p.chunk, p.total);
  bool ok = true;

  if (warp == 0) {
    if (elect_one()) {
      int i = 0, segments = 0;
      for (int t = begin_at; t < end_at; ++t, ++i) {
        const int m = t / p.n_tiles, n = t - m * p.n_tiles;
        if (i == 0 || n == 0) {
          if (!mbar_wait(bar(&ctl->x_empty), (segments & 1) ^ 1, p.dev_status)) { ok = false; break; }
          ++segments;
          mbar_expect_tx(bar(&ctl->x_full), (uint32_t)slices);
          for (int s = 0; s < p.KB; ++s) tma_load_2d(base + x_at + (uint32_t)(s * A_BYTES), &x_map, s * SLICE, m * TILE_M, bar(&ctl->x_full));
        }
        if (!mbar_wait(bar(&ctl->w_empty[i & 1]), ((i >> 1) & 1) ^ 1, p.dev_status)) { ok = false; break; }
        const uint32_t full = bar(&ctl->w_full[i & 1]);
        mbar_expect_tx(full, (uint32_t)slices);
        for (int s = 0; s < p.KB; ++s) tma_load_2d(base + w_at + (uint32_t)((i & 1) * slices + s * A_BYTES), &w_map, s * SLICE, n * TILE_M, full);
      }
      if (!ok) {   // what has been issued lands before the block's shared memory is given back
        if (segments)
          for (int k = 0; k < 100000 && !mbar_try_wait(bar(&ctl->x_full), (uint32_t)((segments - 1) & 1)); ++k) {}
        for (int j = i - 2 < 0 ? 0 : i - 2; j < i; ++j)
          for (int k = 0; k < 100000 && !mbar_try_wait(bar(&ctl->w_full[j & 1]), (uint32_t)((j >> 1) & 1)); ++k) {}
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect_one()) {
      const uint32_t flags = (1u << 4) | ((BF16 ? 1u : 0u) << 7) | ((BF16 ? 1u : 0u) << 10) | ((uint32_t)(TILE_M >> 4) << 24);
      const uint32_t id_s = flags | ((uint32_t)(TILE_M >> 3) << 17), id_dx = flags | (1u << 16) | ((uint32_t)(p.CN >> 3) << 17);
      const uint64_t x_k = smem_desc<128>(base + x_at), w_k = smem_desc<128>(base + w_at), w_mn = smem_desc_mn<128>(base + w_at, A_BYTES), g_k = smem_desc<128>(base + g_at);
      int segments = 0;
      auto logits = [&](int i) {
        const int t = begin_at + i, n = t % p.n_tiles;
        if (i == 0 || n == 0) {
          if (!mbar_wait(bar(&ctl->x_full), segments & 1, p.dev_status)) { ok = false; return; }
          ++segments;
        }
        if (!mbar_wait(bar(&ctl->w_full[i & 1]), (i >> 1) & 1, p.dev_status)) { ok = false; return; }
        tc_fence_after();
        const uint64_t w = w_k + (uint64_t)(((i & 1) * slices) >> 4);
        for (int s = 0; s < p.KB; ++s)
#pragma unroll
          for (int k = 0; k < SLICE / 16; ++k)
            umma_f16(tmem + (uint32_t)((i & 1) * TILE_M), x_k + (uint64_t)((s * A_BYTES) >> 4) + (uint64_t)(k * 2), w + (uint64_t)((s * A_BYTES) >> 4) + (uint64_t)(k * 2), id_s,
                     (s | k) ? 1u : 0u);
        umma_commit(bar(&ctl->s_full[i & 1]));
        if (t + 1 < end_at && n == p.n_tiles - 1) umma_commit(bar(&ctl->x_empty));   // the rows' last logits
      };
      const int count = end_at - begin_at;
      if (count > 0) logits(0);
      int done_segments = 0;
      for (int i = 0; i < count && ok; ++i) {
        if (i + 1 < count) logits(i + 1);                  // (its accumulator was read before g of tile i - 1 was complete)
        if (!ok) break;
        const int n = (begin_at + i) % p.n_tiles;
        const bool opens = i == 0 || n == 0, closes = i + 1 == count || n == p.n_tiles - 1;
        if (!mbar_wait(bar(&ctl->g_full), i & 1, p.dev_status)) { ok = false; break; }
        if (want_x) {
          if (opens && done_segments && !mbar_wait(bar(&ctl->dx_read), (done_segments - 1) & 1, p.dev_status)) { ok = false; break; }
          tc_fence_after();
          const uint64_t w = w_mn + (uint64_t)(((i & 1) * slices) >> 4);
#pragma unroll
          for (int k = 0; k < TILE_M / 16; ++k)
            umma_f16(tmem + dx_col, g_k + (uint64_t)(((k >> 2) * A_BYTES) >> 4) + (uint64_t)((k & 3) * 2), w + (uint64_t)(k * 128), id_dx, (!opens || k) ? 1u : 0u);
        }
        umma_commit(bar(&ctl->w_empty[i & 1]));
        umma_commit(bar(&ctl->g_empty));
        if (want_x && closes) {
          umma_commit(bar(&ctl->dx_full));
          ++done_segments;
        }
      }
      umma_commit(bar(&ctl->done));
      (void)mbar_wait(bar(&ctl->done), 0, p.dev_status);
    }
    __syncwarp();
  } else if (warp == STORE_WARP) {
    if (elect_one()) {
      const int count = end_at - begin_at;
      for (int i = 0; i < count; ++i) {
        if (!mbar_wait(bar(&ctl->g_full), i & 1, p.dev_status)) break;
        if (want_w) {
          void* const to = reinterpret_cast<char*>(p.q.g) + (int64_t)(begin_at + i) * (2 * A_BYTES);
          asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;\n\tcp.async.bulk.commit_group;\n\tcp.async.bulk.wait_group.read 0;" ::"l"(to),
                       "r"(base + (uint32_t)g_at), "r"(2 * A_BYTES)
                       : "memory");
        }
        mbar_arrive(bar(&ctl->g_empty));
      }
      asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    __syncwarp();
  } else {
    const int quarter = warp & 3, part = (warp - ROWS_WARP0) >> 2, in_tile = quarter * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
    const int c_pieces = p.CN / 16, c_first = c_pieces * part / PARTS, c_last = c_pieces * (part + 1) / PARTS;
    RowGrad rg = {};
    int i = 0, segments = 0;
    for (int t = begin_at; t < end_at; ++t, ++i) {
      const int m = t / p.n_tiles, n = t - m * p.n_tiles, row = m * TILE_M + in_tile;
      if (i == 0 || n == 0) rg = row_grad(p.q, row, p.lift);
      if (ok) ok = mbar_wait(bar(&ctl->s_full[i & 1]), (i >> 1) & 1, p.dev_status);
      if (!__all_sync(0xFFFFFFFFu, ok)) { ok = false; break; }
      tc_fence_after();
      {   // 32 of the tile's 128 columns, while g of the tile before is still multiplied
        uint32_t r[32], out[16];
        float z[32];
        const int col = n * TILE_M + part * 32;
        tmem_ld32(lanes + (uint32_t)((i & 1) * TILE_M + part * 32), r);
        tmem_ld_wait();
        to_logits<32>(p.q, r, col, z);
        gradients<32, BF16>(p.q, rg, z, out);
        if (i) ok = mbar_wait(bar(&ctl->g_empty), (i - 1) & 1, p.dev_status);
        if (!__all_sync(0xFFFFFFFFu, ok)) { ok = false; break; }
        uint8_t* const chunk = gen + g_at + (part >> 1) * A_BYTES;
        const int piece = (part & 1) * 4;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          *reinterpret_cast<uint4*>(chunk + tile_offset<128>(in_tile, piece + k)) = make_uint4(out[4 * k], out[4 * k + 1], out[4 * k + 2], out[4 * k + 3]);
        const int in = rg.label - col;
        if (in >= 0 && in < 32)
          reinterpret_cast<uint16_t*>(chunk + tile_offset<128>(in_tile, piece + (in >> 3)))[in & 7] = label_grad<BF16>(p.q, rg, row, p.lift);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(&ctl->g_full));
      if (!want_x || !(t + 1 == end_at || n == p.n_tiles - 1)) continue;
      if (ok) ok = mbar_wait(bar(&ctl->dx_full), segments & 1, p.dev_status);
      ++segments;
      if (!__all_sync(0xFFFFFFFFu, ok)) { ok = false; break; }
      tc_fence_after();
      const int slot = (int)blockIdx.x - m * p.n_tiles / p.chunk;
      float* const to = p.slab + ((int64_t)slot * p.q.rows + row) * p.CN;
      for (int c = c_first; c < c_last; ++c) {
        uint32_t r[16];
        __syncwarp();
        tmem_ld16(lanes + dx_col + (uint32_t)(c * 16), r);
        tmem_ld_wait();
        if (row >= p.q.rows) continue;
        st_global_32B(to + c * 16, r);
        st_global_32B(to + c * 16 + 8, r + 8);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(&ctl->dx_read));
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, 512u);
}

template <auto KERNEL, int BYTES = SMEM_BUDGET> bool allow_smem() {
  static bool configured[64] = {};   // per device
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
  if (!configured[dev]) {
    if (cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, BYTES) != cudaSuccess) {
      (void)cudaGetLastError();
      return false;
    }
    configured[dev] = true;
  }
  return true;
}

int columns_pow2(int cols) {
  int v = 32;
  while (v < cols) v <<= 1;
  return v;
}

// Classes of a tile and how many tiles of a row of them make a unit.
void plan_logits(int rows, int classes, LogitParams* p) {
  p->m_tiles = (rows + TILE_M - 1) / TILE_M;
  p->n_tiles = (classes + 255) / 256;
  p->NT = p->n_tiles <= 4 ? wcn_ce_round((classes + p->n_tiles - 1) / p->n_tiles, 16) : 256;
  // As few rounds of the grid as there can be, counted in tiles; a unit costs the loads of its rows, about a tile.
  const int sms = wcn_num_sms();
  int64_t best = INT64_MAX;
  for (int per = p->n_tiles; per >= 1; --per) {
    const int splits = (p->n_tiles + per - 1) / per;
    if (splits > 64) break;
    const int64_t rounds = ((int64_t)p->m_tiles * splits + sms - 1) / sms, cost = rounds * (per + 1);
    if (cost < best) { best = cost; p->per = per; p->splits = splits; }
  }
  p->units = p->m_tiles * p->splits;
}

template <int RES, bool GRAD, bool BF16>
int launch_logits(LogitParams& p, size_t fixed, cudaStream_t st) {
  const int b_bytes = p.NT * SLICE * 2;
  const int stage = RES == ROWS ? b_bytes : RES == CLASSES ? A_BYTES : A_BYTES + b_bytes;
  const size_t kept = RES == NOTHING ? 0 : (size_t)p.KB * (RES == ROWS ? A_BYTES : b_bytes);
  p.stages = (int)((SMEM_BUDGET - fixed - kept) / stage);
  if (p.stages > MAX_STAGES) p.stages = MAX_STAGES;
  p.tmem_cols = columns_pow2(2 * p.NT);
  CUtensorMap xm, wm;
  if (!matrix_map(&xm, p.q.x, p.q.rows, p.q.channels, p.q.x_ld * 2, TILE_M, BF16) ||
      !matrix_map(&wm, p.q.w, p.q.classes, p.q.channels, p.q.w_ld * 2, p.NT, BF16))
    return WCN_ERR_UNSUPPORTED_CONFIG;
  constexpr auto kern = ce_logits_kernel<RES, GRAD, BF16>;
  if (!allow_smem<kern>()) return WCN_ERR_INITIALIZATION;
  const int sms = wcn_num_sms();
  kern<<<p.units < sms ? p.units : sms, LOGIT_THREADS, fixed + kept + (size_t)p.stages * stage, st>>>(xm, wm, p);
  ++wcn_launched;
  return cudaGetLastError() == cudaSuccess ? WCN_OK : WCN_ERR_EXECUTION;
}

constexpr size_t FIXED = sizeof(Control) + 1024 + 128, FIXED_WHOLE = FIXED + sizeof(WholeRows) + 16;

// Whether the forward kernel finishes the losses: all classes one tile that stays in shared memory.
bool whole_rows(const LogitParams& p) { return p.n_tiles == 1 && p.KB * (int64_t)p.NT * SLICE * 2 + 4 * A_BYTES + (int64_t)FIXED_WHOLE <= SMEM_BUDGET; }

template <bool GRAD, bool BF16> int by_resident(LogitParams& p, cudaStream_t st) {
  const size_t fixed = FIXED;
  const int64_t b_bytes = (int64_t)p.NT * SLICE * 2;
  if (!GRAD && whole_rows(p)) return launch_logits<CLASSES, GRAD, BF16>(p, FIXED_WHOLE, st);
  if (GRAD && p.n_tiles == 1 && p.KB * b_bytes + 4 * A_BYTES + (int64_t)fixed <= SMEM_BUDGET) return launch_logits<CLASSES, GRAD, BF16>(p, fixed, st);
  if (p.KB * (int64_t)A_BYTES + 3 * b_bytes + (int64_t)fixed <= SMEM_BUDGET) return launch_logits<ROWS, GRAD, BF16>(p, fixed, st);
  return launch_logits<NOTHING, GRAD, BF16>(p, fixed, st);
}

// Columns of a tile: with the sums of A's rows beside them.
int most_columns(bool ones) { return ones ? 240 : 256; }

template <bool TRANS, bool BLOCKED, bool BF16>
int launch_product(const wcn_ce_product& q, int32_t* dev_status, cudaStream_t st) {
  constexpr int MB = BLOCKED ? 2 : 1;
  ProductParams p = {};
  p.q = q;
  p.dev_status = dev_status;
  const int most = most_columns(q.slab_ones);
  p.n_tiles = (q.n + most - 1) / most;
  p.NT = wcn_ce_round((q.n + p.n_tiles - 1) / p.n_tiles, 16);
  p.NB = (p.NT + 63) / 64;
  p.m_tiles = (q.m + MB * TILE_M - 1) / (MB * TILE_M);
  p.ksteps = (q.k + SLICE - 1) / SLICE;
  p.per = (p.ksteps + q.splits - 1) / q.splits;
  if ((p.ksteps + p.per - 1) / p.per != q.splits) return WCN_ERR_INVALID_PARAMETERS;
  p.units = p.m_tiles * p.n_tiles * q.splits;
  p.stride = p.NT + (q.slab_ones ? 16 : 0);
  p.accs = 2 * MB * p.stride <= 512 ? 2 : 1;
  p.tmem_cols = columns_pow2(p.accs * MB * p.stride);
  p.vec = q.out && reinterpret_cast<uintptr_t>(q.out) % 32 == 0 && (q.n * 2) % 32 == 0;
  const size_t fixed = sizeof(Control) + 1024 + 128 + SLICE * 128;
  const int stage = MB * A_BYTES + p.NB * SLICE * 128;
  p.stages = (int)((SMEM_BUDGET - fixed) / stage);
  if (p.stages > MAX_STAGES) p.stages = MAX_STAGES;
  CUtensorMap am, bm;
  if (!matrix_map(&bm, q.b, q.k, q.n, q.b_ld * 2, SLICE, BF16)) return WCN_ERR_UNSUPPORTED_CONFIG;
  if (BLOCKED) am = bm;   // (not read)
  else if (!matrix_map(&am, q.a, TRANS ? q.k : q.m, TRANS ? q.m : q.k, q.a_ld * 2, TRANS ? SLICE : TILE_M, BF16)) return WCN_ERR_UNSUPPORTED_CONFIG;
  constexpr auto kern = ce_product_kernel<TRANS, BLOCKED, BF16>;
  if (!allow_smem<kern>()) return WCN_ERR_INITIALIZATION;
  const int sms = wcn_num_sms();
  kern<<<p.units < sms ? p.units : sms, THREADS, fixed + (size_t)p.stages * stage, st>>>(am, bm, p);
  ++wcn_launched;
  return cudaGetLastError() == cudaSuccess ? WCN_OK : WCN_ERR_EXECUTION;
}

// Whether the shapes fit, and how.
bool plan_head(int64_t rows, int channels, int classes, bool bias, HeadParams* p, size_t* smem) {
  if (classes > 256 || channels > 256) return false;
  p->KB = (channels + SLICE - 1) / SLICE;
  p->NT = wcn_ce_round(classes, 16);
  p->CN = wcn_ce_round(channels, 16);
  p->MB = (classes + 127) / 128;
  const int sums = p->MB * (p->CN + (bias ? 16 : 0)), both = p->NT + p->CN, one = p->NT > p->CN ? p->NT : p->CN;
  p->apart = both + sums <= 512;
  p->acc = p->apart ? both : one;
  if (p->acc + sums > 512) return false;
  p->tmem_cols = 512;
  p->tiles = (int)((rows + TILE_M - 1) / TILE_M);
  *smem = 1024 + (size_t)p->KB * p->NT * 128 + 2 * (size_t)p->KB * A_BYTES + (size_t)p->MB * 2 * A_BYTES + ONES_BYTES + sizeof(HeadControl) + 128;
  return *smem <= SMEM_BUDGET;
}

template <bool BF16> int launch_head(HeadParams& p, size_t smem, int blocks, cudaStream_t st) {
  CUtensorMap xm, wm;
  if (!matrix_map(&xm, p.q.x, p.q.rows, p.q.channels, p.q.x_ld * 2, TILE_M, BF16) ||
      !matrix_map(&wm, p.q.w, p.q.classes, p.q.channels, p.q.w_ld * 2, p.NT, BF16))
    return WCN_ERR_UNSUPPORTED_CONFIG;
  constexpr auto kern = ce_head_kernel<BF16>;
  if (!allow_smem<kern>()) return WCN_ERR_INITIALIZATION;
  kern<<<blocks, LOGIT_THREADS, smem, st>>>(xm, wm, p);
  ++wcn_launched;
  return cudaGetLastError() == cudaSuccess ? WCN_OK : WCN_ERR_EXECUTION;
}

size_t rows_smem(int channels) { return 1024 + (size_t)(3 * ((channels + SLICE - 1) / SLICE) + 2) * A_BYTES + sizeof(RowsControl) + 128; }

template <bool BF16> int launch_rows(RowsParams& p, cudaStream_t st) {
  CUtensorMap xm, wm;
  if (!matrix_map(&xm, p.q.x, p.q.rows, p.q.channels, p.q.x_ld * 2, TILE_M, BF16) ||
      !matrix_map(&wm, p.q.w, p.q.classes, p.q.channels, p.q.w_ld * 2, TILE_M, BF16))
    return WCN_ERR_UNSUPPORTED_CONFIG;
  constexpr auto kern = ce_rows_kernel<BF16>;
  if (!allow_smem<kern, ROWS_SMEM>()) return WCN_ERR_INITIALIZATION;
  kern<<<(p.total + p.chunk - 1) / p.chunk, ROWS_THREADS, rows_smem(p.q.channels), st>>>(xm, wm, p);
  ++wcn_launched;
  return cudaGetLastError() == cudaSuccess ? WCN_OK : WCN_ERR_EXECUTION;
}

}  // namespace

// Whether g and dx are one kernel's, and how the (row tile, class tile) pairs of a piece are divided among blocks: `chunk` pairs
// each, so that a row tile has at most `slots` of them.
bool wcn_ce_rows_taken(int channels) { return channels <= 256 && rows_smem(channels) <= (size_t)ROWS_SMEM; }
void wcn_ce_rows_plan(int rows, int classes, int* chunk, int* slots) {
  const int64_t n_tiles = (classes + TILE_M - 1) / TILE_M, total = n_tiles * ((rows + TILE_M - 1) / TILE_M), sms = wcn_num_sms();
  *chunk = (int)((total + sms - 1) / sms);
  *slots = (int)((n_tiles - 1) / *chunk) + 2;
}

int wcn_ce_rows(const wcn_ce_piece& q, float* slab, int dtype, float lift, int32_t* dev_status, cudaStream_t st) {
  RowsParams p = {};
  int slots;
  p.q = q; p.slab = slab; p.lift = lift; p.dev_status = dev_status;
  p.KB = (q.channels + SLICE - 1) / SLICE;
  p.CN = wcn_ce_round(q.channels, 16);
  p.n_tiles = (q.classes + TILE_M - 1) / TILE_M;
  p.total = p.n_tiles * ((q.rows + TILE_M - 1) / TILE_M);
  wcn_ce_rows_plan(q.rows, q.classes, &p.chunk, &slots);
  return dtype == WCN_BF16 ? launch_rows<true>(p, st) : launch_rows<false>(p, st);
}

// Blocks, and with them slabs, of the kernel for few classes; 0: not taken.
int wcn_ce_head_blocks(int64_t rows, int channels, int classes, bool bias) {
  HeadParams p = {};
  size_t smem;
  if (!plan_head(rows, channels, classes, bias, &p, &smem)) return 0;
  const int sms = wcn_num_sms();
  return p.tiles < sms ? p.tiles : sms;
}

int wcn_ce_head(const wcn_ce_piece& q, const wcn_ce_scale& scale, void* dx, float* slab, float* slab_ones, int dtype, float lift,
                int32_t* dev_status, cudaStream_t st) {
  HeadParams p = {};
  size_t smem;
  if (!plan_head(q.rows, q.channels, q.classes, slab_ones, &p, &smem)) return WCN_ERR_UNSUPPORTED_CONFIG;
  p.q = q; p.scale = scale; p.dx = dx; p.slab = slab; p.slab_ones = slab_ones; p.lift = lift; p.dev_status = dev_status;
  p.vec = reinterpret_cast<uintptr_t>(dx) % 32 == 0 && q.channels * 2 % 32 == 0;
  const int sms = wcn_num_sms(), blocks = p.tiles < sms ? p.tiles : sms;
  return dtype == WCN_BF16 ? launch_head<true>(p, smem, blocks, st) : launch_head<false>(p, smem, blocks, st);
}

// Pairs of (largest, sum) that the forward kernel leaves for each row.
int wcn_ce_logits_parts(int rows, int classes) {
  LogitParams p = {};
  plan_logits(rows, classes, &p);
  return p.splits * PARTS;
}

// Blocks of a forward kernel that finishes the losses itself; 0: it leaves parts.
int wcn_ce_whole_blocks(int rows, int classes, int channels) {
  LogitParams p = {};
  p.KB = (channels + SLICE - 1) / SLICE;
  plan_logits(rows, classes, &p);
  const int sms = wcn_num_sms();
  return whole_rows(p) ? (p.units < sms ? p.units : sms) : 0;
}

int wcn_ce_logits(const wcn_ce_piece& q, const wcn_ce_result* out, int dtype, bool gradient, float lift, int32_t* dev_status, cudaStream_t st) {
  LogitParams p = {};
  p.q = q;
  if (out) p.out = *out;
  p.lift = lift;
  p.dev_status = dev_status;
  p.KB = (q.channels + SLICE - 1) / SLICE;
  plan_logits(q.rows, q.classes, &p);
  if (dtype == WCN_BF16) return gradient ? by_resident<true, true>(p, st) : by_resident<false, true>(p, st);
  return gradient ? by_resident<true, false>(p, st) : by_resident<false, false>(p, st);
}

// Splits of k with which the product's tiles keep every multiprocessor busy.
int wcn_ce_product_splits(int m, int n, int k, bool blocked, bool ones) {
  const int tile = blocked ? 2 * TILE_M : TILE_M, most = most_columns(ones), tiles = ((m + tile - 1) / tile) * ((n + most - 1) / most), ksteps = (k + SLICE - 1) / SLICE, sms = wcn_num_sms();
  int best = 1;
  double least = 1e30;
  for (int s = 1; s <= sms && s <= ksteps; ++s) {
    const int per = (ksteps + s - 1) / s;
    if ((ksteps + per - 1) / per != s) continue;
    // rounds of the grid in steps of k, a unit's start and its sums' way out and back counted as some more
    const double cost = (double)((tiles * (int64_t)s + sms - 1) / sms) * (per + 12);
    if (cost < least) { least = cost; best = s; }
  }
  return best;
}

int wcn_ce_product_run(const wcn_ce_product& q, bool transposed, bool blocked, int dtype, int32_t* dev_status, cudaStream_t st) {
  if (blocked) return dtype == WCN_BF16 ? launch_product<true, true, true>(q, dev_status, st) : launch_product<true, true, false>(q, dev_status, st);
  if (dtype == WCN_BF16) return transposed ? launch_product<true, false, true>(q, dev_status, st) : launch_product<false, false, true>(q, dev_status, st);
  return transposed ? launch_product<true, false, false>(q, dev_status, st) : launch_product<false, false, false>(q, dev_status, st);
}
