// Linear layers in fp32 on the tensor cores, with fp32's precision: numbers as sums of three bf16 numbers (split_bf16.cuh), six of the nine
// products of their parts.
//
// A first launch writes the parts of the operands, [3][rows][columns] each.  The second works through tiles of 128 rows x up to 128 columns
// (and, of the weights' gradient, parts of the rows that are summed over): a thread issues TMA loads of 64 of k of all parts into a
// ring, a thread the 24 matrix instructions of such a slice, small products first, into one of several accumulators; sixteen warps add every
// accumulator to sums in their registers (four threads a row), since a tensor core's accumulator cuts what is below its last place
// instead of rounding it, and finish the tile.  A sum that is not finite, for a number that has no parts (infinite, not a number, 2^39 and
// more) or for its size, is made again on the FMA pipes from the numbers as they came.
// Bound by the epilogue and by rounds: 20 000 x 64 -> 256 with SiLU, 314 tiles for 148 multiprocessors, takes 7 us for the parts and 25
// forward, 33 + 18 + 16 for dz, dx and dW, where bytes allow 4 and products 2 each; the bigger 30 000 x 512 -> 256 with GELU 103 both
// launches, 0.46 PFLOP/s of the tensor pipe's products in bf16.
//
// Every wait is bounded (tcgen05_common.cuh); a kernel that gives up sets the status word, waits for its copies and matrix instructions
// and frees its tensor memory; its results, and those of a launch that finds the word set, are NaN.
#include "linear_fp32.cuh"
#include "linear_ce.cuh"
#include "split_bf16.cuh"
#include "tcgen05_common.cuh"
#include "tma_common.cuh"

namespace {

constexpr int TILE_M = 128, MAX_N = 128, SLICE = 64;      // rows, columns of a tile; of k a slice
constexpr int CHUNK = SLICE * 128;                        // 64 of k x 64 columns of an operand whose rows run along k
constexpr int A_PLANE = TILE_M * 128;
constexpr int MAX_STAGES = 4, MAX_ACC = 4;
constexpr int EPI_WARP0 = 2, PARTS = 4, EPI_WARPS = 4 * PARTS, THREADS = (EPI_WARP0 + EPI_WARPS) * 32;
constexpr int SMEM_BUDGET = 226 * 1024;

struct Params {
  wcn_linear_product q;      // (out: of a finished product)
  int64_t a_k, b_k;          // elements from one of k to the next, of A and B as they came; a_ld, b_ld: from row (column) to the next
  float* slab;               // [splits][m][ld]: sums of a part of k, in the place of `out`
  float* slab_ones;          // [splits][m]: of A alone (null: not wanted)
  int NT, m_tiles, n_tiles, ksteps, per, splits, units, stages, accs, stride, tmem_cols, ld;
  int b_plane;
  int vec, vec_bias;         // rows of `out` and of what is added start on 32-byte boundaries; the bias on a 16-byte one
  int32_t* dev_status;
};

struct Ring {
  int slot, phase, depth;
  __device__ __forceinline__ void advance() {
    if (++slot == depth) { slot = 0; phase ^= 1; }
  }
};

struct Control {
  uint64_t full[MAX_STAGES], empty[MAX_STAGES];
  uint64_t acc_full[MAX_ACC], acc_empty[MAX_ACC];
  uint64_t done;
  uint32_t tmem_holder;
  int32_t skip;
};

__device__ __forceinline__ uint32_t bar(uint64_t* b) { return smem_u32(b); }
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}

// Element (row, col) on the FMA pipes, k in order; `ones`: the sum of A's row.
__device__ __noinline__ float again(const wcn_linear_product& q, int64_t a_k, int64_t b_k, int row, int col, int k0, int k1, bool ones) {
  const float* a = (const float*)q.a + (int64_t)row * q.a_ld;
  const float* b = (const float*)q.b + (int64_t)col * q.b_ld;
  float v = 0.f;
  for (int k = k0; k < k1; ++k) v = fmaf(__ldg(a + k * a_k), ones ? 1.f : __ldg(b + k * b_k), v);
  return v;
}

// A_MN, B_MN: rows of A (columns of the result) run along the rows of the operand's matrix, which is [k][m] ([k][n]).  ACT, GRAD: what is
// made of the sums (a kernel for each: one that has all of them waits for its instructions; 20 000 x 64 -> 256 with SiLU, both launches,
// 46 us forward where this takes 33).
template <bool A_MN, bool B_MN, int ACT, bool GRAD>
__global__ void __launch_bounds__(THREADS, 1)
linear_split_kernel(const __grid_constant__ CUtensorMap a_map, const __grid_constant__ CUtensorMap b_map, const __grid_constant__ Params p) {
  extern __shared__ uint8_t smem_raw[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int stage_bytes = 3 * (A_PLANE + p.b_plane);
  const uint32_t pad = ((smem_u32(smem_raw) + 1023u) & ~1023u) - smem_u32(smem_raw), base = smem_u32(smem_raw) + pad;
  uint8_t* const gen = smem_raw + pad + p.stages * stage_bytes;
  const uint32_t ones = base + (uint32_t)(p.stages * stage_bytes);
  const bool with_ones = A_MN && p.slab_ones;
  Control* const ctl = reinterpret_cast<Control*>(gen + (with_ones ? CHUNK : 0));
  const wcn_linear_product& q = p.q;
  auto m_of = [&](int u) { return u / p.n_tiles % p.m_tiles; };
  auto n_of = [&](int u) { return u % p.n_tiles; };
  auto split_of = [&](int u) { return u / (p.n_tiles * p.m_tiles); };
  auto mark = [&]() {
    if (!q.out) return;   // (what joins the sums looks at the status word itself)
    for (int u = blockIdx.x; u < p.units; u += gridDim.x)
      for (int i = threadIdx.x; i < TILE_M * p.NT; i += THREADS) {
        const int row = m_of(u) * TILE_M + i / p.NT, col = n_of(u) * p.NT + i % p.NT;
        if (row < q.m && col < q.n) reinterpret_cast<float*>(q.out)[(int64_t)row * q.out_ld + col] = __int_as_float(0x7FC00000);
      }
  };
  if (threadIdx.x == 0) ctl->skip = *(volatile int32_t*)p.dev_status;
  __syncthreads();
  if (ctl->skip == (int)WCN_ERR_WAIT_EXPIRED) { mark(); return; }
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) { mbar_init(bar(&ctl->full[s]), 1); mbar_init(bar(&ctl->empty[s]), 1); }
    for (int i = 0; i < p.accs; ++i) { mbar_init(bar(&ctl->acc_full[i]), 1); mbar_init(bar(&ctl->acc_empty[i]), EPI_WARPS); }
    mbar_init(bar(&ctl->done), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (with_ones) {   // the sums of A's rows are another 16 columns of the product
    for (int i = threadIdx.x; i < CHUNK / 4; i += THREADS) reinterpret_cast<uint32_t*>(gen)[i] = 0x3F803F80u;
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) tmem_alloc(smem_u32(&ctl->tmem_holder), (uint32_t)p.tmem_cols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctl->tmem_holder;
  bool ok = true;

  if (warp == 0) {
    if (elect_one()) {
      Ring r{0, 0, p.stages};
      int issued = 0;
      for (int u = blockIdx.x; u < p.units && ok; u += gridDim.x) {
        const int m = m_of(u) * TILE_M, n = n_of(u) * p.NT, k0 = split_of(u) * p.per, k1 = min(k0 + p.per, p.ksteps);
        for (int k = k0; k < k1; ++k) {
          if (!mbar_wait(bar(&ctl->empty[r.slot]), r.phase ^ 1, p.dev_status)) { ok = false; break; }
          const uint32_t full = bar(&ctl->full[r.slot]), at = base + (uint32_t)(r.slot * stage_bytes);
          mbar_expect_tx(full, (uint32_t)stage_bytes);
          for (int part = 0; part < 3; ++part) {
            const uint32_t a = at + (uint32_t)(part * A_PLANE), b = at + (uint32_t)(3 * A_PLANE + part * p.b_plane);
            if (A_MN) {
              tma_load_3d(a, &a_map, m, k * SLICE, part, full);
              tma_load_3d(a + CHUNK, &a_map, m + 64, k * SLICE, part, full);
            } else {
              tma_load_3d(a, &a_map, k * SLICE, m, part, full);
            }
            if (B_MN) {
              for (int c = 0; c * CHUNK < p.b_plane; ++c) tma_load_3d(b + (uint32_t)(c * CHUNK), &b_map, n + 64 * c, k * SLICE, part, full);
            } else {
              tma_load_3d(b, &b_map, k * SLICE, n, part, full);
            }
          }
          r.advance();
          ++issued;
        }
      }
      if (!ok)   // what has been issued lands before the block's shared memory is given back
        for (int i = 0; i < issued && i < r.depth; ++i) {
          if (--r.slot < 0) { r.slot = r.depth - 1; r.phase ^= 1; }
          for (int k = 0; k < 100000 && !mbar_try_wait(bar(&ctl->full[r.slot]), (uint32_t)r.phase); ++k) {}
        }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect_one()) {
      const uint32_t flags = (1u << 4) | (1u << 7) | (1u << 10) | (A_MN ? 1u << 15 : 0u) | ((uint32_t)(TILE_M >> 4) << 24);
      const uint32_t idesc = flags | (B_MN ? 1u << 16 : 0u) | ((uint32_t)(p.NT >> 3) << 17), idesc_ones = flags | (1u << 16) | ((uint32_t)(16 >> 3) << 17);
      constexpr int A_STEP = A_MN ? 128 : 2, B_STEP = B_MN ? 128 : 2;   // 16 of k further, in units of 16 bytes
      const uint64_t a0 = A_MN ? smem_desc_mn<128>(base, CHUNK) : smem_desc<128>(base);
      const uint64_t b0 = B_MN ? smem_desc_mn<128>(base + 3 * A_PLANE, CHUNK) : smem_desc<128>(base + 3 * A_PLANE);
      const uint64_t ones0 = smem_desc_mn<128>(ones, CHUNK);
      Ring r{0, 0, p.stages};
      int ab = 0, aphase = 0;
      for (int u = blockIdx.x; u < p.units && ok; u += gridDim.x) {
        const int k0 = split_of(u) * p.per, k1 = min(k0 + p.per, p.ksteps);
        const bool sums = with_ones && n_of(u) == 0;
        for (int k = k0; k < k1; ++k) {
          if (!mbar_wait(bar(&ctl->acc_empty[ab]), aphase ^ 1, p.dev_status) || !mbar_wait(bar(&ctl->full[r.slot]), r.phase, p.dev_status)) { ok = false; break; }
          tc_fence_after();
          const uint64_t slot = (uint64_t)((r.slot * stage_bytes) >> 4);
          const uint32_t d = tmem + (uint32_t)(ab * p.stride);
#pragma unroll
          for (int t = 0; t < 6; ++t) {
            const uint64_t a = a0 + slot + (uint64_t)((split_a(t) * A_PLANE) >> 4), b = b0 + slot + (uint64_t)((split_b(t) * p.b_plane) >> 4);
#pragma unroll
            for (int i = 0; i < SLICE / 16; ++i) umma_f16(d, a + (uint64_t)(i * A_STEP), b + (uint64_t)(i * B_STEP), idesc, (t | i) ? 1u : 0u);
          }
          if (sums)
#pragma unroll
            for (int part = 2; part >= 0; --part)
#pragma unroll
              for (int i = 0; i < SLICE / 16; ++i)
                umma_f16(d + (uint32_t)p.NT, a0 + slot + (uint64_t)(((part * A_PLANE) >> 4) + i * A_STEP), ones0 + (uint64_t)(i * 128), idesc_ones, (part < 2 || i) ? 1u : 0u);
          umma_commit(bar(&ctl->empty[r.slot]));
          umma_commit(bar(&ctl->acc_full[ab]));
          r.advance();
          if (++ab == p.accs) { ab = 0; aphase ^= 1; }
        }
      }
      umma_commit(bar(&ctl->done));
      (void)mbar_wait(bar(&ctl->done), 0, p.dev_status);
    }
    __syncwarp();
  } else {
    const int quarter = warp & 3, part = (warp - EPI_WARP0) >> 2;
    const int pieces = p.NT / 16, first = pieces * part / PARTS, mine = pieces * (part + 1) / PARTS - first;   // of 16 columns, two at most
    int ab = 0, aphase = 0;
    for (int u = blockIdx.x; u < p.units; u += gridDim.x) {
      const int split = split_of(u), k0 = split * p.per, k1 = min(k0 + p.per, p.ksteps), n0 = n_of(u) * p.NT + first * 16;
      const int row = m_of(u) * TILE_M + quarter * 32 + lane;
      const bool live = row < q.m, sums = with_ones && n_of(u) == 0 && part == 0;
      float sum[32], sum_ones = 0.f;
#pragma unroll
      for (int i = 0; i < 32; ++i) sum[i] = 0.f;
      for (int k = k0; k < k1; ++k) {
        if (ok) ok = mbar_wait(bar(&ctl->acc_full[ab]), aphase, p.dev_status);
        if (!__all_sync(0xFFFFFFFFu, ok)) { ok = false; break; }
        tc_fence_after();
        const uint32_t t = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(ab * p.stride);
        uint32_t r0[16], r1[16];
        __syncwarp();
        if (mine > 0) tmem_ld16(t + (uint32_t)(first * 16), r0);
        if (mine > 1) tmem_ld16(t + (uint32_t)((first + 1) * 16), r1);
        tmem_ld_wait();
        if (mine > 0)
#pragma unroll
          for (int i = 0; i < 16; ++i) sum[i] += __uint_as_float(r0[i]);
        if (mine > 1)
#pragma unroll
          for (int i = 0; i < 16; ++i) sum[16 + i] += __uint_as_float(r1[i]);
        if (sums) {
          uint32_t r0[16];
          __syncwarp();
          tmem_ld16(t + (uint32_t)p.NT, r0);
          tmem_ld_wait();
          sum_ones += __uint_as_float(r0[0]);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(&ctl->acc_empty[ab]));
        if (++ab == p.accs) { ab = 0; aphase ^= 1; }
      }
      if (!ok) break;
      if (!live) continue;
      const int from = k0 * SLICE, to = min(k1 * SLICE, q.k);
      if (sums) {
        float v = sum_ones * (1.f / kSplitScale);
        if (!(fabsf(v) < INFINITY)) v = again(q, p.a_k, p.b_k, row, 0, from, to, true);
        p.slab_ones[(int64_t)split * q.m + row] = v;
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        if (c >= mine) continue;
#pragma unroll
        for (int e = 0; e < 16; e += 8) {
          const int col = n0 + c * 16 + e;
          if (col >= (p.slab ? p.ld : q.n)) continue;
          __align__(16) float v[8];
          bool fine = true;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            v[i] = sum[c * 16 + e + i] * kSumScale;
            fine = fine && fabsf(v[i]) < INFINITY;
          }
          if (!fine)
            for (int i = 0; i < 8; ++i)
              if (!(fabsf(v[i]) < INFINITY) && col + i < q.n) v[i] = again(q, p.a_k, p.b_k, row, col + i, from, to, false);
          if (p.slab) {   // (rows of whole 16 columns; B is zero behind the last)
            st_global_32B(p.slab + ((int64_t)split * q.m + row) * p.ld + col, reinterpret_cast<const uint32_t*>(v));
            continue;
          }
          __align__(16) float g[8];
          float* const out = reinterpret_cast<float*>(q.out) + (int64_t)row * q.out_ld + col;
          const float* const add = reinterpret_cast<const float*>(q.add) + (int64_t)row * q.add_ld + col;
          const bool whole = p.vec && col + 8 <= q.n;
          if (q.add) {
            if (whole) {
              *reinterpret_cast<float4*>(g) = __ldg(reinterpret_cast<const float4*>(add));
              *reinterpret_cast<float4*>(g + 4) = __ldg(reinterpret_cast<const float4*>(add) + 1);
            } else {
#pragma unroll
              for (int i = 0; i < 8; ++i) g[i] = col + i < q.n ? __ldg(add + i) : 0.f;
            }
          }
          if (q.bias) {
            __align__(16) float bias[8];
            if (p.vec_bias && col + 8 <= q.n) {
              *reinterpret_cast<float4*>(bias) = __ldg(reinterpret_cast<const float4*>((const float*)q.bias + col));
              *reinterpret_cast<float4*>(bias + 4) = __ldg(reinterpret_cast<const float4*>((const float*)q.bias + col) + 1);
            } else {
#pragma unroll
              for (int i = 0; i < 8; ++i) bias[i] = col + i < q.n ? __ldg((const float*)q.bias + col + i) : 0.f;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] += bias[i];
          }
          float* const dropped = GRAD ? g : v;
          if (!GRAD)
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = activate<ACT>(v[i]);
          if (q.drop.least) {
            float2 t[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) t[i] = make_float2(dropped[2 * i], dropped[2 * i + 1]);
            drop_eight(q.drop, philox_keys(drop_seed(q.drop)), (uint32_t)col / 8, (uint64_t)(q.row0 + row), t);
#pragma unroll
            for (int i = 0; i < 4; ++i) { dropped[2 * i] = t[i].x; dropped[2 * i + 1] = t[i].y; }
          }
          if (GRAD) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = through<ACT>(g[i], v[i]);
          } else if (q.add) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] += g[i];
          }
          if (whole) {
            st_global_32B(out, reinterpret_cast<const uint32_t*>(v));
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (col + i < q.n) out[i] = v[i];
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

// ------------------------------------------------------------------ parts

struct SplitMatrix {
  const float* x;
  char* planes;            // [3][rows][pitch] bf16
  int64_t rows, ld;
  int cols, across;        // across: pieces of eight of a row
  int vec;                 // rows start on 16-byte boundaries
  unsigned blocks;
};
struct SplitList {
  SplitMatrix m[3];
};

constexpr int SPLIT_THREADS = 256, SPLIT_PIECES = 4;   // pieces of eight numbers a thread

__global__ void __launch_bounds__(SPLIT_THREADS) linear_parts_kernel(const __grid_constant__ SplitList list) {
  unsigned block = blockIdx.x;
  int at = 0;
  while (at < 2 && block >= list.m[at].blocks) { block -= list.m[at].blocks; ++at; }
  const SplitMatrix& s = list.m[at];
  const int64_t pitch = (int64_t)s.across * 8, pieces = s.rows * s.across;
#pragma unroll
  for (int j = 0; j < SPLIT_PIECES; ++j) {
    const int64_t i = ((int64_t)block * SPLIT_PIECES + j) * SPLIT_THREADS + threadIdx.x;
    if (i >= pieces) continue;
    const int64_t row = i / s.across;
    const int col = (int)(i - row * s.across) * 8;
    const float* const x = s.x + row * s.ld + col;
    float v[8];
    if (s.vec && col + 8 <= s.cols) {
      const float4 a = __ldg(reinterpret_cast<const float4*>(x)), b = __ldg(reinterpret_cast<const float4*>(x) + 1);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = col + e < s.cols ? __ldg(x + e) : 0.f;
    }
    store_parts(v, s.planes + (row * pitch + col) * 2, s.rows * pitch * 2);
  }
}

// ------------------------------------------------------------------ host

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

bool parts_map(CUtensorMap* map, const void* planes, int64_t rows, int64_t cols, int box_rows) {
  EncodeTiledFn encode = encode_tiled();
  if (!encode) return false;
  const cuuint64_t pitch = (cuuint64_t)((cols + 7) / 8 * 16);
  const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, 3};
  const cuuint64_t strides[2] = {pitch, pitch * (cuuint64_t)rows};
  const cuuint32_t box[3] = {64u, (cuuint32_t)box_rows, 1u};
  const cuuint32_t step[3] = {1, 1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(planes), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int columns_of(int n) {
  const int tiles = (n + MAX_N - 1) / MAX_N;
  return wcn_ce_round((n + tiles - 1) / tiles, 16);
}

template <bool A_MN, bool B_MN, int ACT, bool GRAD> int launch(Params& p, const void* a_planes, const void* b_planes, cudaStream_t st) {
  const wcn_linear_product& q = p.q;
  p.NT = columns_of(q.n);
  p.m_tiles = (q.m + TILE_M - 1) / TILE_M;
  p.n_tiles = (q.n + p.NT - 1) / p.NT;
  p.ksteps = (q.k + SLICE - 1) / SLICE;
  p.per = (p.ksteps + p.splits - 1) / p.splits;
  if ((p.ksteps + p.per - 1) / p.per != p.splits) return WCN_ERR_INVALID_PARAMETERS;
  p.units = p.m_tiles * p.n_tiles * p.splits;
  p.ld = wcn_ce_round(q.n, 16);
  p.b_plane = B_MN ? (p.NT + 63) / 64 * CHUNK : p.NT * 128;
  p.stride = p.NT + (p.slab_ones ? 16 : 0);
  p.accs = 512 / p.stride < MAX_ACC ? 512 / p.stride : MAX_ACC;
  p.tmem_cols = 32;
  while (p.tmem_cols < p.accs * p.stride) p.tmem_cols *= 2;
  auto boundary = [](const void* at, int64_t ld) { return !at || (reinterpret_cast<uintptr_t>(at) % 32 == 0 && ld % 8 == 0); };
  p.vec = boundary(q.out, q.out_ld) && boundary(q.add, q.add_ld);
  p.vec_bias = reinterpret_cast<uintptr_t>(q.bias) % 16 == 0;
  const int fixed = 1024 + (int)sizeof(Control) + 64 + (p.slab_ones ? CHUNK : 0), stage = 3 * (A_PLANE + p.b_plane);
  p.stages = (SMEM_BUDGET - fixed) / stage;
  if (p.stages > MAX_STAGES) p.stages = MAX_STAGES;
  CUtensorMap a, b;
  const bool ok = (A_MN ? parts_map(&a, a_planes, q.k, q.m, SLICE) : parts_map(&a, a_planes, q.m, q.k, TILE_M)) &&
                  (B_MN ? parts_map(&b, b_planes, q.k, q.n, SLICE) : parts_map(&b, b_planes, q.n, q.k, p.NT));
  if (!ok) return WCN_ERR_UNSUPPORTED_CONFIG;
  constexpr auto kern = linear_split_kernel<A_MN, B_MN, ACT, GRAD>;
  if (!allow_smem<kern>()) return WCN_ERR_INITIALIZATION;
  const int sms = wcn_num_sms();
  kern<<<(unsigned)(p.units < sms ? p.units : sms), THREADS, (size_t)fixed + (size_t)p.stages * stage, st>>>(a, b, p);
  ++wcn_launched;
  return cudaGetLastError() == cudaSuccess ? WCN_OK : WCN_ERR_EXECUTION;
}

}  // namespace

// Bytes of the parts of a matrix.
int64_t wcn_linear_parts_bytes(int64_t rows, int cols) { return (rows * ((cols + 7) / 8 * 8) * 6 + 127) / 128 * 128; }

// The parts of up to three matrices in one launch.
int wcn_linear_parts(const wcn_linear_matrix* m, int count, cudaStream_t st) {
  SplitList list = {};
  unsigned blocks = 0;
  for (int i = 0; i < count; ++i) {
    SplitMatrix& s = list.m[i];
    s.x = m[i].x; s.planes = (char*)m[i].planes; s.rows = m[i].rows; s.ld = m[i].ld; s.cols = m[i].cols; s.across = (m[i].cols + 7) / 8;
    s.vec = reinterpret_cast<uintptr_t>(s.x) % 16 == 0 && s.ld % 4 == 0;
    s.blocks = (unsigned)((s.rows * s.across + SPLIT_THREADS * SPLIT_PIECES - 1) / (SPLIT_THREADS * SPLIT_PIECES));
    blocks += s.blocks;
  }
  linear_parts_kernel<<<blocks, SPLIT_THREADS, 0, st>>>(list);
  ++wcn_launched;
  return cudaGetLastError() == cudaSuccess ? WCN_OK : WCN_ERR_EXECUTION;
}

// A finished product of operands whose parts are made (by_k: B is [k][n]).
int wcn_linear_split(const wcn_linear_product& q, bool by_k, const void* a_planes, const void* b_planes, int32_t* dev_status, cudaStream_t st) {
  Params p = {};
  p.q = q;
  p.a_k = 1;
  p.b_k = 1;
  p.splits = 1;
  p.dev_status = dev_status;
  if (!by_k) {
    switch (q.act) {
      case WCN_ACT_RELU: return q.grad ? launch<false, false, WCN_ACT_RELU, true>(p, a_planes, b_planes, st) : launch<false, false, WCN_ACT_RELU, false>(p, a_planes, b_planes, st);
      case WCN_ACT_SILU: return q.grad ? launch<false, false, WCN_ACT_SILU, true>(p, a_planes, b_planes, st) : launch<false, false, WCN_ACT_SILU, false>(p, a_planes, b_planes, st);
      case WCN_ACT_GELU: return q.grad ? launch<false, false, WCN_ACT_GELU, true>(p, a_planes, b_planes, st) : launch<false, false, WCN_ACT_GELU, false>(p, a_planes, b_planes, st);
      default: return launch<false, false, WCN_ACT_NONE, false>(p, a_planes, b_planes, st);   // (its gradient asks for no z)
    }
  }
  p.q.b_ld = 1;
  p.b_k = q.b_ld;
  return launch<false, true, WCN_ACT_NONE, false>(p, a_planes, b_planes, st);
}

// The sums of parts of the rows of a [k][m] and b [k][n]: a^T b, and those of a.
int wcn_linear_split_weight(const wcn_ce_product& c, const void* a_planes, const void* b_planes, int32_t* dev_status, cudaStream_t st) {
  Params p = {};
  p.q.a = c.a; p.q.b = c.b; p.q.m = c.m; p.q.n = c.n; p.q.k = c.k;
  p.q.a_ld = p.q.b_ld = 1;
  p.a_k = c.a_ld;
  p.b_k = c.b_ld;
  p.slab = c.slab;
  p.slab_ones = c.slab_ones;
  p.splits = c.splits;
  p.dev_status = dev_status;
  return launch<true, true, WCN_ACT_NONE, false>(p, a_planes, b_planes, st);
}

// Parts of the rows with which the tiles keep every multiprocessor busy.
int wcn_linear_split_splits(int m, int n, int k) {
  const int tiles = ((m + TILE_M - 1) / TILE_M) * ((n + columns_of(n) - 1) / columns_of(n)), ksteps = (k + SLICE - 1) / SLICE, sms = wcn_num_sms();
  int best = 1;
  double least = 1e30;
  for (int s = 1; s <= sms && s <= ksteps; ++s) {
    const int per = (ksteps + s - 1) / s;
    if ((ksteps + per - 1) / per != s) continue;
    const double cost = (double)((tiles * (int64_t)s + sms - 1) / sms) * (per + 4);   // rounds of the grid in slices, a unit's start and end as some more
    if (cost < least) { least = cost; best = s; }
  }
  return best;
}
