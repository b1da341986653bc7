// The gradients of a narrow linear layer in 16 bits in one kernel, the gradient behind the activation never in global memory:
//     dz = dropout'(dy) act'(x W^T + bias),   dx = dz W,   dW = dz^T x,   dbias = column sums of dz.
//
// Per 128 rows and 64 outputs: z on the tensor cores; sixteen epilogue warps make dz of it and of dy, in place where TMA has brought dy
// (two halves of 64 outputs are worked on by eight warps each, in turns); with 128 outputs of dz, dx += dz W and dW += dz^T x.  The
// accumulators of dW, all outputs x inputs, stay in tensor memory until the block's last tile, beside those of dx and two of z: 128 +
// inputs (1 + outputs / 128) of 512 columns.  The same images in shared memory serve every product: a tile of rows whose columns run
// along 128-byte (or, for inputs that are no multiple of 64, 64-byte) lines is a K-major operand with its rows on the M / N side, or an
// MN-major one with its rows on the K side.  Sums of the blocks are joined by linear.cu.
// The column sums are made of dz before it is rounded, by exchanges among the lanes.  A launch has 8192 rows a block at most (linear.cu).
// 240 000 x 96 -> 384 bf16 with GELU 120 us (277 MB at 2.3 TB/s; z, dz, dx and dW in launches of their own took 190), without
// activation 79, with dropout 175: the time is the slope's and the generator's, a piece of a warp after the other; the tensor pipe waits
// for dz.
//
// Every wait is bounded (tcgen05_common.cuh); a kernel that gives up sets the status word, waits for its copies and matrix instructions
// and frees its tensor memory; its results, and those of a launch that finds the word set, are NaN (dW and dbias: where they are joined).
#include "linear_16bit.cuh"
#include "linear_ce.cuh"
#include "tma_common.cuh"

namespace {

constexpr int TILE_M = 128, CHUNK_N = 128;                // rows of a tile; outputs of a chunk
constexpr int HALF_BYTES = TILE_M * 128;                  // 64 outputs of dy
constexpr int EPI_WARP0 = 2, PARTS = 4, EPI_WARPS = 4 * PARTS, THREADS = (EPI_WARP0 + EPI_WARPS) * 32;
constexpr int Z_COLUMNS = 128, MAX_BUFFERS = 4;            // buffers: chunks of dy in shared memory
constexpr int SMEM_BUDGET = 226 * 1024;

struct Params {
  wcn_linear_product q;     // a: x [m][k], b: W [n][k], add: dy [m][n]; out: dx [m][k] (null: not wanted)
  float* slab;              // [blocks][n][ld] (null: not wanted)
  float* slab_ones;         // [blocks][n] (null: not wanted)
  int KS, K16, NB, ld;      // slices of k, columns of dx and dW, chunks of outputs
  int tiles, vec, buffers;
  int32_t* dev_status;
};

struct Ring {
  int slot, phase, depth;
  __device__ __forceinline__ void advance() {
    if (++slot == depth) { slot = 0; phase ^= 1; }
  }
};

struct Control {
  uint64_t w_full, x_full[2], x_empty[2], dy_full[MAX_BUFFERS], dz_full[MAX_BUFFERS], dz_empty[MAX_BUFFERS], z_full[2], z_empty[2], dx_full, dx_read, acc_full, done;
  uint32_t tmem_holder;
  int32_t skip;
  PhiloxKeys keys;
};

// The sums over the warp's rows of 16 columns: each pair of lanes has one column's.
__device__ __forceinline__ float column_sums(const float2 (&v)[8], int lane, int& column) {
  float a[8], b[4], c[2];
  const bool h = lane & 16, q = lane & 8, e = lane & 4, s = lane & 2;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 low = v[i], high = v[i + 4];
    a[2 * i] = (h ? high.x : low.x) + __shfl_xor_sync(0xFFFFFFFFu, h ? low.x : high.x, 16);
    a[2 * i + 1] = (h ? high.y : low.y) + __shfl_xor_sync(0xFFFFFFFFu, h ? low.y : high.y, 16);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) b[i] = (q ? a[i + 4] : a[i]) + __shfl_xor_sync(0xFFFFFFFFu, q ? a[i] : a[i + 4], 8);
#pragma unroll
  for (int i = 0; i < 2; ++i) c[i] = (e ? b[i + 2] : b[i]) + __shfl_xor_sync(0xFFFFFFFFu, e ? b[i] : b[i + 2], 4);
  float d = (s ? c[1] : c[0]) + __shfl_xor_sync(0xFFFFFFFFu, s ? c[0] : c[1], 2);
  d += __shfl_xor_sync(0xFFFFFFFFu, d, 1);
  column = (h ? 8 : 0) + (q ? 4 : 0) + (e ? 2 : 0) + (s ? 1 : 0);
  return d;
}

// RB: bytes of a line of x and W (64 or 32 inputs).
template <int ACT, int RB, bool BF16>
__global__ void __launch_bounds__(THREADS, 1)
linear_backward_kernel(const __grid_constant__ CUtensorMap x_map, const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap dy_map,
                       const __grid_constant__ Params p) {
  extern __shared__ uint8_t smem_raw[];
  constexpr int DEPTH = RB / 2;                            // inputs of a slice
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int w_slice = p.NB * CHUNK_N * RB, x_slice = TILE_M * RB, x_stage = p.KS * x_slice;
  const uint32_t pad = ((smem_u32(smem_raw) + 1023u) & ~1023u) - smem_u32(smem_raw), base = smem_u32(smem_raw) + pad;
  const uint32_t w_at = base, x_at = w_at + (uint32_t)(p.KS * w_slice), dy_at = x_at + (uint32_t)(2 * x_stage), end_at = dy_at + (uint32_t)(p.buffers * 2 * HALF_BYTES);
  uint8_t* const gen = smem_raw + pad;
  float* const sums = reinterpret_cast<float*>(gen + (end_at - base));                         // [4][NB * 128]
  float* const biases = sums + (p.slab_ones ? 4 * p.NB * CHUNK_N : 0);                          // [NB * 128]
  Control* const ctl = reinterpret_cast<Control*>(biases + p.NB * CHUNK_N);
  const wcn_linear_product& q = p.q;
  const int halves = (q.n + 63) / 64;
  const bool with_z = ACT != WCN_ACT_NONE;
  auto mark = [&]() {
    if (!q.out) return;
    const uint16_t nan = BF16 ? 0x7FC0 : 0x7E00;
    for (int t = blockIdx.x; t < p.tiles; t += gridDim.x)
      for (int i = threadIdx.x; i < TILE_M * q.k; i += THREADS) {
        const int row = t * TILE_M + i / q.k;
        if (row < q.m) reinterpret_cast<uint16_t*>(q.out)[(int64_t)row * q.out_ld + i % q.k] = nan;
      }
  };
  if (threadIdx.x == 0) ctl->skip = *(volatile int32_t*)p.dev_status;
  __syncthreads();
  if (ctl->skip == (int)WCN_ERR_WAIT_EXPIRED) { mark(); return; }
  if (threadIdx.x == 0) {
    mbar_init(bar(&ctl->w_full), 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(&ctl->x_full[i]), 1);
      mbar_init(bar(&ctl->x_empty[i]), 1);
      mbar_init(bar(&ctl->z_full[i]), 1);
      mbar_init(bar(&ctl->z_empty[i]), EPI_WARPS / 2);
    }
    for (int i = 0; i < p.buffers; ++i) {
      mbar_init(bar(&ctl->dy_full[i]), 1);
      mbar_init(bar(&ctl->dz_full[i]), EPI_WARPS);
      mbar_init(bar(&ctl->dz_empty[i]), 1);
    }
    mbar_init(bar(&ctl->dx_full), 1);
    mbar_init(bar(&ctl->dx_read), EPI_WARPS);
    mbar_init(bar(&ctl->acc_full), 1);
    mbar_init(bar(&ctl->done), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  for (int i = threadIdx.x; i < p.NB * CHUNK_N; i += THREADS) {
    biases[i] = q.bias && i < q.n ? number<BF16>(reinterpret_cast<const uint16_t*>(q.bias)[i]) : 0.f;
    if (p.slab_ones)
      for (int s = 0; s < 4; ++s) sums[s * p.NB * CHUNK_N + i] = 0.f;
  }
  if (threadIdx.x == 32 && q.drop.least) ctl->keys = philox_keys(drop_seed(q.drop));
  if (warp == 1) tmem_alloc(smem_u32(&ctl->tmem_holder), 512u);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctl->tmem_holder;
  const uint32_t dx_col = tmem + (uint32_t)(with_z ? Z_COLUMNS : 0), dw_col = dx_col + (uint32_t)p.K16;
  bool ok = true;

  if (warp == 0) {
    if (elect_one()) {
      mbar_expect_tx(bar(&ctl->w_full), (uint32_t)(p.KS * w_slice));
      for (int s = 0; s < p.KS; ++s)
        for (int j = 0; j < p.NB; ++j) tma_load_2d(w_at + (uint32_t)(s * w_slice + j * CHUNK_N * RB), &w_map, s * DEPTH, j * CHUNK_N, bar(&ctl->w_full));
      int i = 0, chunks = 0;  // so far
      Ring g{0, 0, p.buffers};
      for (int t = blockIdx.x; t < p.tiles && ok; t += gridDim.x, ++i) {
        if (!mbar_wait(bar(&ctl->x_empty[i & 1]), ((i >> 1) & 1) ^ 1, p.dev_status)) { ok = false; break; }
        mbar_expect_tx(bar(&ctl->x_full[i & 1]), (uint32_t)x_stage);
        for (int s = 0; s < p.KS; ++s) tma_load_2d(x_at + (uint32_t)((i & 1) * x_stage + s * x_slice), &x_map, s * DEPTH, t * TILE_M, bar(&ctl->x_full[i & 1]));
        for (int j = 0; j < p.NB; ++j) {
          if (!mbar_wait(bar(&ctl->dz_empty[g.slot]), g.phase ^ 1, p.dev_status)) { ok = false; break; }
          const uint32_t full = bar(&ctl->dy_full[g.slot]), to = dy_at + (uint32_t)(g.slot * 2 * HALF_BYTES);
          const bool two = 2 * j + 1 < halves;
          mbar_expect_tx(full, (uint32_t)(two ? 2 * HALF_BYTES : HALF_BYTES));
          tma_load_2d(to, &dy_map, j * CHUNK_N, t * TILE_M, full);
          if (two) tma_load_2d(to + HALF_BYTES, &dy_map, j * CHUNK_N + 64, t * TILE_M, full);
          g.advance();
          ++chunks;
        }
      }
      if (!ok) {   // what has been issued lands before the block's shared memory is given back
        for (int k = 0; k < 100000 && !mbar_try_wait(bar(&ctl->w_full), 0); ++k) {}
        for (int v = i - 2 < 0 ? 0 : i - 2; v < i; ++v)
          for (int k = 0; k < 100000 && !mbar_try_wait(bar(&ctl->x_full[v & 1]), (uint32_t)((v >> 1) & 1)); ++k) {}
        for (int v = 0; v < chunks && v < g.depth; ++v) {
          if (--g.slot < 0) { g.slot = g.depth - 1; g.phase ^= 1; }
          for (int k = 0; k < 100000 && !mbar_try_wait(bar(&ctl->dy_full[g.slot]), (uint32_t)g.phase); ++k) {}
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect_one()) {
      const uint32_t flags = (1u << 4) | ((BF16 ? 1u : 0u) << 7) | ((BF16 ? 1u : 0u) << 10) | ((uint32_t)(TILE_M >> 4) << 24);
      const uint32_t idesc_z = flags | ((uint32_t)(64 >> 3) << 17);
      const uint32_t idesc_dx = flags | (1u << 16) | ((uint32_t)(p.K16 >> 3) << 17), idesc_dw = idesc_dx | (1u << 15);
      const uint64_t w_k = smem_desc<RB>(w_at), w_mn = smem_desc_mn<RB>(w_at, (uint32_t)w_slice);
      const uint64_t x_k = smem_desc<RB>(x_at), x_mn = smem_desc_mn<RB>(x_at, (uint32_t)x_slice);
      const uint64_t dz_k = smem_desc<128>(dy_at), dz_mn = smem_desc_mn<128>(dy_at, HALF_BYTES);
      constexpr int LINES = 16 * RB / 16;                  // 16 lines of x or W further, in units of 16 bytes
      int i = 0;
      uint32_t zs = 0;       // parities of the two accumulators' uses
      Ring g{0, 0, p.buffers};
      ok = mbar_wait(bar(&ctl->w_full), 0, p.dev_status);
      for (int t = blockIdx.x; t < p.tiles && ok; t += gridDim.x, ++i) {
        const uint64_t x_stage_at = (uint64_t)(((i & 1) * x_stage) >> 4);
        if (!mbar_wait(bar(&ctl->x_full[i & 1]), (i >> 1) & 1, p.dev_status)) { ok = false; break; }
        tc_fence_after();
        auto issue_z = [&](int h) {   // 64 outputs
          if (!mbar_wait(bar(&ctl->z_empty[h & 1]), (zs >> (h & 1) & 1) ^ 1, p.dev_status)) return false;
          zs ^= 1u << (h & 1);
          tc_fence_after();
          for (int s = 0; s < p.KS; ++s)
#pragma unroll
            for (int e = 0; e < DEPTH / 16; ++e)
              umma_f16(tmem + (uint32_t)((h & 1) * 64), x_k + x_stage_at + (uint64_t)(((s * x_slice) >> 4) + e * 2),
                       w_k + (uint64_t)(((s * w_slice + h * 64 * RB) >> 4) + e * 2), idesc_z, (s | e) ? 1u : 0u);
          umma_commit(bar(&ctl->z_full[h & 1]));
          return true;
        };
        auto products = [&](int j) {  // of 128 outputs of dz
          if (!mbar_wait(bar(&ctl->dz_full[g.slot]), g.phase, p.dev_status)) return false;
          if (j == 0 && i > 0 && q.out && !mbar_wait(bar(&ctl->dx_read), (i - 1) & 1, p.dev_status)) return false;
          tc_fence_after();
          const uint64_t at = (uint64_t)((g.slot * 2 * HALF_BYTES) >> 4);
          if (q.out) {
            const int here = min(2, halves - 2 * j);
            for (int h = 0; h < here; ++h)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                umma_f16(dx_col, dz_k + at + (uint64_t)((h * HALF_BYTES >> 4) + e * 2), w_mn + (uint64_t)(((j * CHUNK_N + h * 64) * RB >> 4) + e * LINES), idesc_dx,
                         (j | h | e) ? 1u : 0u);
          }
          if (p.slab)
#pragma unroll
            for (int e = 0; e < TILE_M / 16; ++e)
              umma_f16(dw_col + (uint32_t)(j * p.K16), dz_mn + at + (uint64_t)(e * 128), x_mn + x_stage_at + (uint64_t)(e * LINES), idesc_dw, (i | e) ? 1u : 0u);
          umma_commit(bar(&ctl->dz_empty[g.slot]));
          g.advance();
          return true;
        };
        for (int j = 0; j < p.NB && ok; ++j) {
          if (with_z) {
            ok = issue_z(2 * j);
            if (ok && 2 * j + 1 < halves) ok = issue_z(2 * j + 1);
          }
          if (ok && j > 0) ok = products(j - 1);
        }
        if (ok) ok = products(p.NB - 1);
        if (!ok) break;
        if (q.out) umma_commit(bar(&ctl->dx_full));
        umma_commit(bar(&ctl->x_empty[i & 1]));
      }
      umma_commit(bar(&ctl->acc_full));
      umma_commit(bar(&ctl->done));
      (void)mbar_wait(bar(&ctl->done), 0, p.dev_status);
    }
    __syncwarp();
  } else {
    const int quarter = warp & 3, part = (warp - EPI_WARP0) >> 2, side = part >> 1, col_half = part & 1;   // side: which half of 64 outputs; which 32 of them
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const int in_tile = quarter * 32 + lane;
    uint32_t place[4];                       // this thread's 32 outputs of its row of dy
#pragma unroll
    for (int c = 0; c < 4; ++c) place[c] = dy_at + (uint32_t)(side * HALF_BYTES + in_tile * 128 + (((col_half * 4 + c) ^ (in_tile & 7)) << 4));
    int i = 0, zs = 0;
    Ring g{0, 0, p.buffers};
    for (int t = blockIdx.x; t < p.tiles; t += gridDim.x, ++i) {
      const int row = t * TILE_M + in_tile;
      for (int j = 0; j < p.NB; ++j, g.advance()) {
        const bool use = 2 * j + side < halves;
        if (ok) ok = mbar_wait(bar(&ctl->dy_full[g.slot]), g.phase, p.dev_status);
        if (ok && with_z && use) ok = mbar_wait(bar(&ctl->z_full[side]), zs & 1, p.dev_status);
        if (!__all_sync(0xFFFFFFFFu, ok)) { ok = false; break; }
        if (use) {
          uint32_t r[32];
          if (with_z) {
            ++zs;
            tc_fence_after();
            tmem_ld32(tmem + lanes + (uint32_t)(side * 64 + col_half * 32), r);
            tmem_ld_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(&ctl->z_empty[side]));
          }
          const int col = j * CHUNK_N + side * 64 + col_half * 32;
          const uint32_t buffer = (uint32_t)(g.slot * 2 * HALF_BYTES);
          const float4* const bias = reinterpret_cast<const float4*>(biases + col);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint4 add[2];
            add[0] = load_shared(place[2 * h] + buffer);
            add[1] = load_shared(place[2 * h + 1] + buffer);
            float2 v[8];
            if (with_z) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float4 b = bias[4 * h + e];
                v[2 * e] = __fadd2_rn(make_float2(__uint_as_float(r[16 * h + 4 * e]), __uint_as_float(r[16 * h + 4 * e + 1])), make_float2(b.x, b.y));
                v[2 * e + 1] = __fadd2_rn(make_float2(__uint_as_float(r[16 * h + 4 * e + 2]), __uint_as_float(r[16 * h + 4 * e + 3])), make_float2(b.z, b.w));
              }
            }
            finish<ACT, true, BF16, true>(q, &ctl->keys, v, add, q.row0 + row, col + 16 * h);
            if (with_z || q.drop.least) {   // (otherwise dy is dz)
              store_shared(place[2 * h] + buffer, make_uint4(pack2<BF16>(v[0]), pack2<BF16>(v[1]), pack2<BF16>(v[2]), pack2<BF16>(v[3])));
              store_shared(place[2 * h + 1] + buffer, make_uint4(pack2<BF16>(v[4]), pack2<BF16>(v[5]), pack2<BF16>(v[6]), pack2<BF16>(v[7])));
            }
            if (p.slab_ones) {
              int column;
              const float sum = column_sums(v, lane, column);
              if (!(lane & 1)) sums[quarter * p.NB * CHUNK_N + col + 16 * h + column] += sum;   // (this warp's columns alone)
            }
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(&ctl->dz_full[g.slot]));
      }
      if (!ok) break;
      if (q.out) {
        ok = mbar_wait(bar(&ctl->dx_full), i & 1, p.dev_status);
        if (!__all_sync(0xFFFFFFFFu, ok)) { ok = false; break; }
        tc_fence_after();
        uint16_t* const out = reinterpret_cast<uint16_t*>(q.out) + (int64_t)row * q.out_ld;
        for (int c = part; c * 16 < p.K16; c += PARTS) {
          uint32_t r[16];
          __syncwarp();
          tmem_ld16(dx_col + lanes + (uint32_t)(c * 16), r);
          tmem_ld_wait();
          if (row >= q.m) continue;
          uint32_t v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = pack2<BF16>(__fmul2_rn(make_float2(__uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1])), both(q.factor)));
          if (p.vec && c * 16 + 16 <= q.k) {
            st_global_32B(out + c * 16, v);
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (c * 16 + e < q.k) out[c * 16 + e] = (uint16_t)(v[e / 2] >> (16 * (e & 1)));
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(&ctl->dx_read));
      }
    }
    if (p.slab && ok) {   // this block's sums
      ok = mbar_wait(bar(&ctl->acc_full), 0, p.dev_status);
      if (__all_sync(0xFFFFFFFFu, ok)) {
        tc_fence_after();
        for (int j = 0; j < p.NB; ++j)
          for (int c = part; c * 16 < p.K16; c += PARTS) {
            uint32_t r[16];
            __syncwarp();
            tmem_ld16(dw_col + lanes + (uint32_t)(j * p.K16 + c * 16), r);
            tmem_ld_wait();
            const int n = j * CHUNK_N + in_tile;
            if (n >= q.n) continue;
            float* const to = p.slab + ((int64_t)blockIdx.x * q.n + n) * p.ld + c * 16;
            st_global_32B(to, r);
            st_global_32B(to + 8, r + 8);
          }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, 512u);
  if (p.slab_ones)
    for (int n = threadIdx.x; n < q.n; n += THREADS) {
      const int all = p.NB * CHUNK_N;
      p.slab_ones[(int64_t)blockIdx.x * q.n + n] = (sums[n] + sums[all + n]) + (sums[2 * all + n] + sums[3 * all + n]);
    }
  if (threadIdx.x == 0) ctl->skip = *(volatile int32_t*)p.dev_status;
  __syncthreads();
  if (ctl->skip == (int)WCN_ERR_WAIT_EXPIRED) mark();
}

// ------------------------------------------------------------------ host

int line_bytes(int k) { return k % 64 == 0 || k % 64 > 32 ? 128 : 64; }

// Whether the shapes fit, and how.
bool plan(int k, int n, bool with_z, bool sums, Params* p, size_t* smem) {
  const int rb = line_bytes(k);
  p->KS = (k * 2 + rb - 1) / rb;
  p->K16 = wcn_ce_round(k, 16);
  p->ld = p->K16;
  p->NB = (n + CHUNK_N - 1) / CHUNK_N;
  if (k > 256 || (with_z ? Z_COLUMNS : 0) + p->K16 * (p->NB + 1) > 512) return false;
  const size_t rest = 1024 + (size_t)p->KS * p->NB * CHUNK_N * rb + 2 * (size_t)p->KS * TILE_M * rb + (size_t)(sums ? 5 : 1) * p->NB * CHUNK_N * 4 + sizeof(Control) + 64;   // (what stands before Control is a multiple of 16 bytes)
  for (p->buffers = MAX_BUFFERS; p->buffers >= 2; --p->buffers) {   // dy is on its way for as many chunks
    *smem = rest + (size_t)p->buffers * 2 * HALF_BYTES;
    if (*smem <= SMEM_BUDGET) return true;
  }
  return false;
}

template <auto KERNEL> bool allow_smem() {
  static bool configured[64] = {};   // per device
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
  if (!configured[dev]) {
    if (cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BUDGET) != cudaSuccess) {
      (void)cudaGetLastError();
      return false;
    }
    configured[dev] = true;
  }
  return true;
}

template <int RB> bool lines_map(EncodeTiledFn encode, CUtensorMap* map, bool bf16, const void* base, int64_t rows, int64_t cols, int64_t ld) {
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)(ld * 2)};
  const cuuint32_t box[2] = {RB / 2, TILE_M};
  const cuuint32_t step[2] = {1, 1};
  return encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(base), dims, strides, box, step,
                CU_TENSOR_MAP_INTERLEAVE_NONE, RB == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int ACT, int RB, bool BF16> int launch(const Params& p, size_t smem, int blocks, cudaStream_t st) {
  const wcn_linear_product& q = p.q;
  EncodeTiledFn encode = encode_tiled();
  if (!encode) return WCN_ERR_UNSUPPORTED_CONFIG;
  CUtensorMap x, w, dy;
  if (!lines_map<RB>(encode, &x, BF16, q.a, q.m, q.k, q.a_ld) || !lines_map<RB>(encode, &w, BF16, q.b, q.n, q.k, q.b_ld) ||
      !lines_map<128>(encode, &dy, BF16, q.add, q.m, q.n, q.add_ld))
    return WCN_ERR_UNSUPPORTED_CONFIG;
  constexpr auto kern = linear_backward_kernel<ACT, RB, BF16>;
  if (!allow_smem<kern>()) return WCN_ERR_INITIALIZATION;
  kern<<<(unsigned)blocks, THREADS, smem, st>>>(x, w, dy, p);
  ++wcn_launched;
  return cudaGetLastError() == cudaSuccess ? WCN_OK : WCN_ERR_EXECUTION;
}

template <int RB, bool BF16> int by_act(const Params& p, size_t smem, int blocks, cudaStream_t st) {
  switch (p.q.act) {
    case WCN_ACT_RELU: return launch<WCN_ACT_RELU, RB, BF16>(p, smem, blocks, st);
    case WCN_ACT_SILU: return launch<WCN_ACT_SILU, RB, BF16>(p, smem, blocks, st);
    case WCN_ACT_GELU: return launch<WCN_ACT_GELU, RB, BF16>(p, smem, blocks, st);
    default: return launch<WCN_ACT_NONE, RB, BF16>(p, smem, blocks, st);
  }
}

}  // namespace

// Blocks, and with them parts of the sums, of the kernel that makes all gradients of `rows` rows; 0: not taken.
int wcn_linear_backward_blocks(int64_t rows, int k, int n, int act, bool sums) {
  Params p = {};
  size_t smem;
  if (!plan(k, n, act != WCN_ACT_NONE, sums, &p, &smem)) return 0;
  const int64_t tiles = (rows + TILE_M - 1) / TILE_M, sms = wcn_num_sms();
  return (int)(tiles < sms ? tiles : sms);
}

// q: x, W, bias and dy as linear.cuh has them for dz (`out`: dx); slab [blocks][n][k rounded up to 16], slab_ones [blocks][n].  Rows of x, W and
// dy start on 16-byte boundaries.
int wcn_linear_backward_run(const wcn_linear_product& q, float* slab, float* slab_ones, bool bf16, int32_t* dev_status, cudaStream_t st) {
  Params p = {};
  size_t smem;
  if (!plan(q.k, q.n, q.act != WCN_ACT_NONE, slab_ones, &p, &smem)) return WCN_ERR_UNSUPPORTED_CONFIG;
  p.q = q; p.slab = slab; p.slab_ones = slab_ones; p.dev_status = dev_status;
  p.tiles = (q.m + TILE_M - 1) / TILE_M;
  p.vec = reinterpret_cast<uintptr_t>(q.out) % 32 == 0 && q.out_ld % 16 == 0;
  const int sms = wcn_num_sms(), blocks = p.tiles < sms ? p.tiles : sms;
  if (line_bytes(q.k) == 128) return bf16 ? by_act<128, true>(p, smem, blocks, st) : by_act<128, false>(p, smem, blocks, st);
  return bf16 ? by_act<64, true>(p, smem, blocks, st) : by_act<64, false>(p, smem, blocks, st);
}
