// Linear layers in 16 and 8 bits on the tensor cores: out = add + dropout(act(A B^T + bias)), and what their gradients need of the
// same form (see linear.cuh).
//
// Persistent blocks work through tiles of 128 rows x NT columns (up to 256): one thread issues TMA tile loads into a ring, one the
// matrix instructions (fp32 accumulators in tensor memory, as many tiles as fit), sixteen warps empty them.  Each of those takes 32 rows x 32
// columns at a time, in turns over the tile's columns and over tiles: bias, activation, dropout and the addition are made in
// registers in fp32 and the sum is rounded once.  What is added (the residual, or the gradient that arrives) comes by TMA into the warp's
// own 2 KB of shared memory, one piece ahead, and the result leaves from the same place by TMA: rows of 64 bytes per thread
// would cost the load/store pipe a line each.  Rows that TMA cannot take (pitches that are no multiple of 16 bytes) go the same way
// through shared memory and from there in elements.
// Where they fit beside a ring of four tiles, the columns' rows of B stay in shared memory: a block then has one group of
// columns, and A alone passes.  Elsewhere, with 192 columns of a tile and six slices of k and more, two blocks of a cluster share a tile of 256
// rows (one instruction for both, B's rows halved between them): half of B's bytes from L2, which bound the wide layers.
//
// Sixteen warps empty the accumulators: with eight, twelve and 24 the layer below took 98, 82 and 78 us where it takes 72.
// 240 000 rows, bf16, us: 96 -> 384 40 (5.7 TB/s), with GELU 65, with dropout too 117.  GELU is some 270 arithmetic instructions of 430 for a
// warp's 32 x 32 numbers; issue slots are 60 % busy and HBM half: a warp has one piece at a time and waits between its load from tensor
// memory and its store.  The generator is as many instructions again.  384 -> 96 with residual 46 (6.0 TB/s).
// 60 000 x 256 -> 1 024 with GELU 82, its dz 95 to 100, its dx 40.  100 000 x 1 024 -> 1 024 of 8 bits 99 (2.1 PFLOP/s), with SiLU and
// residual 113 to 118.
//
// Every wait is bounded (tcgen05_common.cuh); a kernel that gives up sets the status word, waits for its copies and matrix instructions
// and frees its tensor memory; its results, and those of a launch that finds the word set, are NaN.
#include "linear_16bit.cuh"
#include "tma_common.cuh"

namespace {

constexpr int TILE_M = 128, SLICE_BYTES = 128;             // rows of a tile; bytes of k of a stage
constexpr int A_BYTES = TILE_M * SLICE_BYTES;
constexpr int MN_CHUNK = 64 * 128;                         // 64 of k x 64 columns of a B whose columns run along its rows
constexpr int MAX_STAGES = 12, MAX_ACC = 8;
constexpr int EPI_WARP0 = 2, PARTS = 4, EPI_WARPS = 4 * PARTS, THREADS = (EPI_WARP0 + EPI_WARPS) * 32;
constexpr int PIECE = 32, PIECE_BYTES = 32 * PIECE * 2;    // columns of a warp's piece; its 32 rows in shared memory
constexpr int LASTING = 1024;                              // columns whose bias is kept
constexpr int SMEM_BUDGET = 226 * 1024;

struct Params {
  wcn_linear_product q;
  int KB, NT;               // slices of k; columns of a tile (a multiple of 32)
  int m_tiles, n_tiles, stages, accs, tmem_cols;
  int b_slice;              // bytes of a slice of B
  int out_tma, add_tma, resident, pair;
  int wide, turns;          // pieces of a warp's turn, turns of a tile
  int lasting;              // bias and scales are in shared memory from the start on: of the block's columns, or of all
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
  uint64_t b_full;
  uint64_t acc_full[MAX_ACC], acc_empty[MAX_ACC];
  uint64_t add_full[EPI_WARPS][2];
  uint64_t done;
  uint32_t tmem_holder;
  int32_t skip;
  PhiloxKeys keys;
  __align__(16) float bias[LASTING], scale[LASTING];   // of all columns that this block has, or of each warp's piece
};

__device__ __forceinline__ void umma_f8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// What two blocks of a cluster do together (PAIR): one matrix instruction has 256 rows, of which each block holds 128, and half of the
// columns' rows of B from each.
__device__ __forceinline__ uint32_t of_block(uint32_t at, uint32_t rank) {   // the same place in the shared memory of a block of the cluster
  uint32_t there;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(at), "r"(rank));
  return there;
}
__device__ __forceinline__ void arrive_at(uint32_t there) { asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(there) : "memory"); }
__device__ __forceinline__ void store_at(uint32_t there, int32_t v) { asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(there), "r"(v) : "memory"); }
__device__ __forceinline__ void cluster_meet() { asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar_of_first) {
  asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar_of_first)
               : "memory");
}
__device__ __forceinline__ void umma_pair_f16(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_pair_f8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void commit_pair(uint32_t bar) {   // the barriers at this place in both blocks
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
}
__device__ __forceinline__ void tmem_alloc_pair(uint32_t holder, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(holder), "r"(cols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, int x, int y, uint32_t src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(src)
               : "memory");
}
__device__ __forceinline__ void store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void store_wait_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory"); }

// The tiles of a block.  With the columns' rows of B in shared memory: one group of columns, a part of its tiles of rows; else all tiles
// in order, columns fastest.
template <bool PAIR> struct Tiles {
  int m, n, dm, dn, m_tiles, n_tiles;
  __device__ __forceinline__ explicit Tiles(const Params& p) : m_tiles(p.m_tiles), n_tiles(p.n_tiles) {
    const int grid = PAIR ? (int)gridDim.x / 2 : (int)gridDim.x, block = PAIR ? (int)blockIdx.x / 2 : (int)blockIdx.x;
    m = block / n_tiles;
    n = block - m * n_tiles;
    dm = p.resident ? (grid - n + n_tiles - 1) / n_tiles : grid / n_tiles;   // (resident: the blocks of this group)
    dn = p.resident ? 0 : grid - dm * n_tiles;
  }
  __device__ __forceinline__ bool there() const { return m < m_tiles; }
  __device__ __forceinline__ void advance() {
    m += dm;
    n += dn;
    if (n >= n_tiles) { n -= n_tiles; ++m; }
  }
};

// KIND: operands f16, bf16 or e4m3.  B_MN: the columns of the result run along B's rows.
// ACT, GRAD: what is made of the sums (see linear.cuh); a kernel for each, as one that has all of them waits for its instructions.
template <int KIND, bool B_MN, int ACT, bool GRAD, bool BF16, bool PAIR>
__global__ void __launch_bounds__(THREADS, 1)
linear_kernel(const __grid_constant__ CUtensorMap a_map, const __grid_constant__ CUtensorMap b_map, const __grid_constant__ CUtensorMap out_map,
              const __grid_constant__ CUtensorMap add_map, const __grid_constant__ Params p) {
  extern __shared__ uint8_t smem_raw[];
  constexpr int DEPTH = KIND == WCN_E4M3 ? 128 : 64;       // elements of k of a slice
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int TILE_ROWS = PAIR ? 2 * TILE_M : TILE_M;
  const int rank = PAIR ? (int)blockIdx.x & 1 : 0, row_of_block = rank * TILE_M;
  const bool resident = !PAIR && p.resident;
  const int stage_bytes = resident ? A_BYTES : A_BYTES + p.b_slice;
  const uint32_t pad = ((smem_u32(smem_raw) + 1023u) & ~1023u) - smem_u32(smem_raw);
  const uint32_t base = smem_u32(smem_raw) + pad;
  const uint32_t res = base + (uint32_t)(p.stages * stage_bytes), staging = res + (resident ? (uint32_t)(p.KB * p.b_slice) : 0u);
  uint8_t* const staging_at = smem_raw + (staging - smem_u32(smem_raw));
  Control* const ctl = reinterpret_cast<Control*>(staging_at + EPI_WARPS * 2 * PIECE_BYTES);
  const wcn_linear_product& q = p.q;
  uint16_t* const out = reinterpret_cast<uint16_t*>(q.out);
  auto mark = [&]() {
    const uint16_t nan = BF16 ? 0x7FC0 : 0x7E00;
    for (Tiles<PAIR> t(p); t.there(); t.advance())
      for (int i = threadIdx.x; i < TILE_M * p.NT; i += THREADS) {
        const int row = t.m * TILE_ROWS + row_of_block + i / p.NT, col = t.n * p.NT + i % p.NT;
        if (row < q.m && col < q.n) out[(int64_t)row * q.out_ld + col] = nan;
      }
  };
  if (!PAIR) {
    if (threadIdx.x == 0) ctl->skip = *(volatile int32_t*)p.dev_status;
    __syncthreads();
  } else {   // (one answer for both blocks, which are both there)
    cluster_meet();
    if (threadIdx.x == 0 && rank == 0) {
      const int32_t status = *(volatile int32_t*)p.dev_status;
      ctl->skip = status;
      store_at(of_block(smem_u32(&ctl->skip), 1), status);
    }
    cluster_meet();
  }
  if (ctl->skip == (int)WCN_ERR_WAIT_EXPIRED) { mark(); return; }
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) { mbar_init(bar(&ctl->full[s]), 1); mbar_init(bar(&ctl->empty[s]), 1); }
    mbar_init(bar(&ctl->b_full), 1);
    for (int i = 0; i < p.accs; ++i) { mbar_init(bar(&ctl->acc_full[i]), 1); mbar_init(bar(&ctl->acc_empty[i]), (uint32_t)(4 * p.turns * (PAIR ? 2 : 1))); }
    for (int w = 0; w < EPI_WARPS; ++w)
      for (int i = 0; i < 2; ++i) mbar_init(bar(&ctl->add_full[w][i]), 1);
    mbar_init(bar(&ctl->done), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (threadIdx.x == 32 && q.drop.least) ctl->keys = philox_keys(drop_seed(q.drop));
  if (p.lasting && !B_MN) {
    const int first = resident ? (int)blockIdx.x % p.n_tiles * p.NT : 0;
    for (int i = threadIdx.x; i < p.lasting; i += THREADS) {
      const bool there = first + i < q.n;
      ctl->bias[i] = q.bias && there ? number<BF16>(reinterpret_cast<const uint16_t*>(q.bias)[first + i]) : 0.f;
      if (KIND == WCN_E4M3) ctl->scale[i] = there ? __ldg(&q.b_scale[first + i]) : 0.f;
    }
  }
  if (warp == 1) {
    if (PAIR) tmem_alloc_pair(smem_u32(&ctl->tmem_holder), (uint32_t)p.tmem_cols);
    else tmem_alloc(smem_u32(&ctl->tmem_holder), (uint32_t)p.tmem_cols);
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_meet();   // (barriers are there before the other block reaches for them)
  tc_fence_after();
  const uint32_t tmem = ctl->tmem_holder;
  bool ok = true;

  if (warp == 0) {
    if (elect_one()) {
      Ring r{0, 0, p.stages};
      int issued = 0;
      auto load = [&](uint32_t to, const CUtensorMap* map, int x, int y, uint32_t full) {
        if (PAIR) tma_load_pair(to, map, x, y, full);
        else tma_load_2d(to, map, x, y, full);
      };
      auto load_b = [&](uint32_t to, int s, int n, uint32_t full) {   // (PAIR: this block's half of the columns)
        const int col = n * p.NT + (PAIR ? rank * (p.NT / 2) : 0);
        if (B_MN) {
          for (int c = 0; c * MN_CHUNK < p.b_slice; ++c) load(to + (uint32_t)(c * MN_CHUNK), &b_map, col + 64 * c, s * DEPTH, full);
        } else {
          load(to, &b_map, s * DEPTH, col, full);
        }
      };
      Tiles<PAIR> t(p);
      const bool any = t.there();
      if (resident && any) {
        mbar_expect_tx(bar(&ctl->b_full), (uint32_t)(p.KB * p.b_slice));
        for (int s = 0; s < p.KB; ++s) load_b(res + (uint32_t)(s * p.b_slice), s, t.n, bar(&ctl->b_full));
      }
      for (; t.there() && ok; t.advance())
        for (int s = 0; s < p.KB; ++s) {
          if (!mbar_wait(bar(&ctl->empty[r.slot]), r.phase ^ 1, p.dev_status)) { ok = false; break; }
          // (PAIR: the first block's barrier counts what both receive)
          const uint32_t full = PAIR ? of_block(bar(&ctl->full[r.slot]), 0) : bar(&ctl->full[r.slot]), at = base + (uint32_t)(r.slot * stage_bytes);
          if (rank == 0) mbar_expect_tx(bar(&ctl->full[r.slot]), (uint32_t)(PAIR ? 2 * stage_bytes : stage_bytes));
          load(at, &a_map, s * DEPTH, t.m * TILE_ROWS + row_of_block, full);
          if (!resident) load_b(at + A_BYTES, s, t.n, full);
          r.advance();
          ++issued;
        }
      if (!ok && rank) {   // (whose copies the first block's barriers count: time for them to land)
        for (const long long began = clock64(); clock64() - began < 2000000ll;) {}
      } else if (!ok) {   // what has been issued lands before the block's shared memory is given back
        for (int i = 0; i < issued && i < r.depth; ++i) {
          if (--r.slot < 0) { r.slot = r.depth - 1; r.phase ^= 1; }
          for (int k = 0; k < 100000 && !mbar_try_wait(bar(&ctl->full[r.slot]), (uint32_t)r.phase); ++k) {}
        }
        for (int k = 0; resident && any && k < 100000 && !mbar_try_wait(bar(&ctl->b_full), 0); ++k) {}
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0 && elect_one()) {
      constexpr uint32_t type = KIND == WCN_BF16 ? 1u : 0u;   // (f16 and e4m3: 0 of their kinds)
      const uint32_t idesc = (1u << 4) | (type << 7) | (type << 10) | (B_MN ? 1u << 16 : 0u) | ((uint32_t)(p.NT >> 3) << 17) | ((uint32_t)(TILE_ROWS >> 4) << 24);
      constexpr int B_STEP = B_MN ? 128 : 2;                  // an instruction's depth further, in units of 16 bytes
      auto describe_b = [&](uint32_t at) { return B_MN ? smem_desc_mn<128>(at, MN_CHUNK) : smem_desc<128>(at); };
      const uint64_t a0 = smem_desc<128>(base), b0 = describe_b(resident ? res : base + A_BYTES);
      Ring r{0, 0, p.stages};
      int ab = 0, aphase = 0;
      Tiles<PAIR> t(p);
      if (resident && t.there()) ok = mbar_wait(bar(&ctl->b_full), 0, p.dev_status);
      for (; ok && t.there(); t.advance()) {
        if (!mbar_wait(bar(&ctl->acc_empty[ab]), aphase ^ 1, p.dev_status)) { ok = false; break; }
        tc_fence_after();
        const uint32_t d = tmem + (uint32_t)(ab * p.NT);
        for (int s = 0; s < p.KB; ++s) {
          if (!mbar_wait(bar(&ctl->full[r.slot]), r.phase, p.dev_status)) { ok = false; break; }
          tc_fence_after();
          const uint64_t slot = (uint64_t)((r.slot * stage_bytes) >> 4);
          const uint64_t a = a0 + slot, b = b0 + (resident ? (uint64_t)((s * p.b_slice) >> 4) : slot);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (PAIR && KIND == WCN_E4M3) umma_pair_f8(d, a + (uint64_t)(i * 2), b + (uint64_t)(i * B_STEP), idesc, (s | i) ? 1u : 0u);
            else if (PAIR) umma_pair_f16(d, a + (uint64_t)(i * 2), b + (uint64_t)(i * B_STEP), idesc, (s | i) ? 1u : 0u);
            else if (KIND == WCN_E4M3) umma_f8(d, a + (uint64_t)(i * 2), b + (uint64_t)(i * B_STEP), idesc, (s | i) ? 1u : 0u);
            else umma_f16(d, a + (uint64_t)(i * 2), b + (uint64_t)(i * B_STEP), idesc, (s | i) ? 1u : 0u);
          }
          if (PAIR) commit_pair(bar(&ctl->empty[r.slot]));
          else umma_commit(bar(&ctl->empty[r.slot]));
          r.advance();
        }
        if (!ok) break;
        if (PAIR) commit_pair(bar(&ctl->acc_full[ab]));
        else umma_commit(bar(&ctl->acc_full[ab]));
        if (++ab == p.accs) { ab = 0; aphase ^= 1; }
      }
      if (PAIR) commit_pair(bar(&ctl->done));
      else umma_commit(bar(&ctl->done));
      (void)mbar_wait(bar(&ctl->done), 0, p.dev_status);
    }
    __syncwarp();
  } else {
    // A warp takes one piece at a time where something is added, else two side by side (what a turn costs besides is then shared).
    // Turns of the block's tiles are numbered through, columns fastest; a warp has every PARTS-th.  It has then seen the accumulator's
    // last tile but one filled (of tiles of one, two .. turns there are 8, 4 .. accumulators at least), as waits by parity want.
    const int ew = warp - EPI_WARP0, quarter = warp & 3, pieces = p.NT / PIECE, wide = p.wide, turns = p.turns;
    uint8_t* const mine = staging_at + ew * 2 * PIECE_BYTES;
    const uint32_t mine_at = staging + (uint32_t)(ew * 2 * PIECE_BYTES);
    const int rows = q.m - row_of_block - quarter * 32, step = p.NT;    // of this warp's quarters: there is one to do where a tile's first row is less
    struct Place {
      int row, n, turn, ab, phase;                       // first row of the tile, its place among the columns' tiles
    };
    const Tiles<PAIR> first(p);
    const int dm = first.dm * TILE_ROWS, dn = first.dn, end = p.m_tiles * TILE_ROWS;
    auto next = [&](Place& w) {
      w.turn += PARTS;
      while (w.turn >= turns) {
        w.turn -= turns;
        w.row += dm;
        w.n += dn;
        if (w.n >= p.n_tiles) { w.n -= p.n_tiles; w.row += TILE_ROWS; }
        if (++w.ab == p.accs) { w.ab = 0; w.phase ^= 1; }
      }
    };
    auto col_of = [&](const Place& w) { return w.n * step + w.turn * wide * PIECE; };
    const bool added = GRAD || q.add, by_tma = added && p.add_tma, more = GRAD ? q.drop.least != 0 : added || q.drop.least;
    auto request = [&](const Place& w, int buffer) {   // one lane
      const uint32_t full = bar(&ctl->add_full[ew][buffer]);
      mbar_expect_tx(full, PIECE_BYTES);
      tma_load_2d(mine_at + (uint32_t)(buffer * PIECE_BYTES), &add_map, col_of(w), w.row + row_of_block + quarter * 32, full);
    };
    Place now{first.m * TILE_ROWS, first.n, (ew >> 2) - PARTS, 0, 0};
    next(now);
    int b = 0;                               // the next piece's place in shared memory
    uint32_t pending = 0, phases = 0;        // of each of the two: whether a copy is on its way there, its barrier's phase
    if (by_tma && now.row < end && now.row < rows && col_of(now) < q.n) {
      if (lane == 0) request(now, 0);
      pending = 1;
    }
    const float factor = q.factor;
    uint32_t swizzled[4];                    // this lane's row of a piece, 16 bytes at a time
#pragma unroll
    for (int c = 0; c < 4; ++c) swizzled[c] = mine_at + (uint32_t)(lane * 64 + ((c ^ (lane >> 1 & 3)) << 4));
    while (now.row < end) {
      Place then = now;
      next(then);
      const int col0 = col_of(now), row0 = now.row + row_of_block + quarter * 32, row = row0 + lane;
      const bool use = now.row < rows && col0 < q.n;
      const float row_scale = KIND == WCN_E4M3 && use && row < q.m ? __ldg(&q.a_scale[row]) : 0.f;
      // What the last turn has left has been read from its place, which is this one's or the next copy's.
      const bool ask = by_tma && then.row < end && then.row < rows && col_of(then) < q.n;
      const int other = use ? b ^ 1 : b;
      if (lane == 0) {
        store_wait_read<0>();
        if (ask) request(then, other);
      }
      if (ask) pending |= 1u << other;
      if (!p.lasting && !B_MN && use)
        for (int j = 0; j < wide; ++j) {
          const int col = col0 + j * PIECE + lane, at = (ew * 2 + j) * PIECE + lane;
          ctl->bias[at] = q.bias && col < q.n ? number<BF16>(reinterpret_cast<const uint16_t*>(q.bias)[col]) : 0.f;
          if (KIND == WCN_E4M3) ctl->scale[at] = col < q.n ? __ldg(&q.b_scale[col]) : 0.f;
        }
      __syncwarp();
      auto element = [&](int line, int c) { return reinterpret_cast<uint16_t*>(mine + b * PIECE_BYTES + line * 64 + (((c >> 3) ^ (line >> 1 & 3)) << 4) + (c & 7) * 2); };
      if (added && use) {
        if (by_tma) {
          if (ok) ok = mbar_wait(bar(&ctl->add_full[ew][b]), phases >> b & 1, p.dev_status);
          if (!__all_sync(0xFFFFFFFFu, ok)) { ok = false; break; }
          phases ^= 1u << b;
          pending &= ~(1u << b);
        } else {
          for (int l = 0; l < 32; ++l)
            *element(l, lane) = row0 + l < q.m && col0 + lane < q.n ? reinterpret_cast<const uint16_t*>(q.add)[(int64_t)(row0 + l) * q.add_ld + col0 + lane] : (uint16_t)0;
          __syncwarp();
        }
      }
      if (ok) ok = mbar_wait(bar(&ctl->acc_full[now.ab]), now.phase, p.dev_status);
      if (!__all_sync(0xFFFFFFFFu, ok)) { ok = false; break; }
      tc_fence_after();
      const uint32_t taddr = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(now.ab * step);
      const int last = min(now.turn * wide + wide, pieces) - 1;
#pragma unroll 1
      for (int piece = now.turn * wide, col = col0; piece <= last; ++piece, col += PIECE) {
        uint32_t r[32];
        tmem_ld32(taddr + (uint32_t)(piece * PIECE), r);
        tmem_ld_wait();
        if (piece == last) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (PAIR && rank) arrive_at(of_block(bar(&ctl->acc_empty[now.ab]), 0));
            else mbar_arrive(bar(&ctl->acc_empty[now.ab]));
          }
        }
        if (!use || col >= q.n) continue;
        const int kept = p.lasting ? (resident ? piece * PIECE : col) : (ew * 2 + piece - now.turn * wide) * PIECE;
        const float4* const bias = reinterpret_cast<const float4*>(ctl->bias + kept);
        const float4* const scale = reinterpret_cast<const float4*>(ctl->scale + kept);
        const uint32_t place = (uint32_t)(b * PIECE_BYTES);
#pragma unroll
        for (int h = 0; h < 2; ++h) {   // (half a piece at a time, for the registers)
          float2 v[8];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            v[2 * i] = make_float2(__uint_as_float(r[16 * h + 4 * i]), __uint_as_float(r[16 * h + 4 * i + 1]));
            v[2 * i + 1] = make_float2(__uint_as_float(r[16 * h + 4 * i + 2]), __uint_as_float(r[16 * h + 4 * i + 3]));
            if (B_MN) {
              v[2 * i] = __fmul2_rn(v[2 * i], both(factor));
              v[2 * i + 1] = __fmul2_rn(v[2 * i + 1], both(factor));
              continue;
            }
            const float4 t = bias[4 * h + i];
            if (KIND == WCN_E4M3) {
              const float4 s = scale[4 * h + i];
              v[2 * i] = __ffma2_rn(__fmul2_rn(v[2 * i], both(row_scale)), make_float2(s.x, s.y), make_float2(t.x, t.y));
              v[2 * i + 1] = __ffma2_rn(__fmul2_rn(v[2 * i + 1], both(row_scale)), make_float2(s.z, s.w), make_float2(t.z, t.w));
            } else {
              v[2 * i] = __fadd2_rn(v[2 * i], make_float2(t.x, t.y));
              v[2 * i + 1] = __fadd2_rn(v[2 * i + 1], make_float2(t.z, t.w));
            }
          }
          uint4 add[2];
          if (added) {
            add[0] = load_shared(swizzled[2 * h] + place);
            add[1] = load_shared(swizzled[2 * h + 1] + place);
          }
          if (more) finish<ACT, GRAD, BF16, true>(q, &ctl->keys, v, add, q.row0 + row, col + 16 * h);
          else finish<ACT, GRAD, BF16, false>(q, &ctl->keys, v, add, q.row0 + row, col + 16 * h);
#pragma unroll
          for (int c = 0; c < 2; ++c)
            store_shared(swizzled[2 * h + c] + place, make_uint4(pack2<BF16>(v[4 * c]), pack2<BF16>(v[4 * c + 1]), pack2<BF16>(v[4 * c + 2]), pack2<BF16>(v[4 * c + 3])));
        }
        if (p.out_tma) {
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&out_map, col, row0, mine_at + place);
            store_commit();
          }
        } else {
          __syncwarp();
          for (int l = 0; l < 32; ++l)
            if (row0 + l < q.m && col + lane < q.n) out[(int64_t)(row0 + l) * q.out_ld + col + lane] = *element(l, lane);
          if (by_tma) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // (the next copy of what is added comes to this place)
          __syncwarp();
        }
        b ^= 1;
      }
      now = then;
    }
    // what is still on its way to or from this warp's places
    for (int i = 0; i < 2; ++i)
      for (int k = 0; (pending >> i & 1) && k < 100000 && !mbar_try_wait(bar(&ctl->add_full[ew][i]), phases >> i & 1); ++k) {}
    if (lane == 0) store_wait_read<0>();
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) {   // (neither block's memory goes while the other one's instructions may reach for it)
    cluster_meet();
    if (warp == 1) tmem_dealloc_pair(tmem, (uint32_t)p.tmem_cols);
  } else if (warp == 1) {
    tmem_dealloc(tmem, (uint32_t)p.tmem_cols);
  }
  if (threadIdx.x == 0) ctl->skip = *(volatile int32_t*)p.dev_status;
  __syncthreads();
  if (ctl->skip == (int)WCN_ERR_WAIT_EXPIRED) {
    asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");   // (results on their way are written before what replaces them)
    __syncthreads();
    mark();
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

// A row-major matrix of `size`-byte elements read or written in boxes of cols x rows, swizzled over their row's bytes (64 or 128).
bool box_map(EncodeTiledFn encode, CUtensorMap* map, CUtensorMapDataType type, int size, const void* base, int64_t rows, int64_t cols, int64_t ld, int box_cols, int box_rows) {
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)(ld * size)};
  const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows};
  const cuuint32_t step[2] = {1, 1};
  return encode(map, type, 2, const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                box_cols * size == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool tma_rows(const void* p, int64_t ld, int size) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * size % 16 == 0; }

constexpr int FIXED = 1024 + EPI_WARPS * 2 * PIECE_BYTES + (int)sizeof(Control) + 64;

// Columns of a tile, and whether B's stay in shared memory.
void plan(const wcn_linear_product& q, int kind, bool b_mn, Params* p) {
  const int depth = kind == WCN_E4M3 ? 128 : 64, sms = wcn_num_sms();
  p->KB = (q.k + depth - 1) / depth;
  p->m_tiles = (q.m + TILE_M - 1) / TILE_M;
  auto slice = [&](int nt) { return b_mn ? (nt + 63) / 64 * MN_CHUNK : nt * SLICE_BYTES; };
  auto tiles_of = [&](int nt) { return (q.n + nt - 1) / nt; };
  auto even = [&](int most) {   // columns of a tile when as few as can be of `most` at the most share them
    const int tiles = tiles_of(most);
    return ((q.n + tiles - 1) / tiles + PIECE - 1) / PIECE * PIECE;
  };
  bool resident = false;
  int nt = even(256);
  for (int most = 256; most >= 128 && !resident; most -= 64) {
    const int t = even(most);
    if ((int64_t)p->KB * slice(t) + 4 * A_BYTES + FIXED <= SMEM_BUDGET && tiles_of(t) * 4 <= sms) { resident = true; nt = t; }
  }
  // few tiles: narrower ones, for as many multiprocessors
  while (nt > PIECE && (int64_t)p->m_tiles * tiles_of(nt) * 2 <= sms) nt = even((nt / 2 + PIECE - 1) / PIECE * PIECE);
  if (!resident || tiles_of(nt) * 4 > sms) resident = (int64_t)p->KB * slice(nt) + 4 * A_BYTES + FIXED <= SMEM_BUDGET && (int64_t)p->m_tiles * tiles_of(nt) <= sms;
  p->NT = nt;
  p->n_tiles = tiles_of(nt);
  p->b_slice = slice(nt);
  p->accs = 512 / nt < MAX_ACC ? 512 / nt : MAX_ACC;
  // Operands that both pass: two blocks share a tile of 256 rows, each with half of B's rows, where there are tiles for all of them.
  // What arrives in a block's shared memory is then 64 bytes a clock of the matrix instructions; alone, 96 at 256 columns, it waits.
  // 100 000 rows bf16, a block a tile and two, us: 1 024 -> 1 024 198, 163; 1 024 -> 256 73, 67; 768 -> 256 60, 54; 384 -> 256 38, 36; 512 -> 200
  // 46, 40; of 8-bit operands 1 024 -> 1 024 118, 99; 768 -> 256 (six slices) 40, 38.  Narrower tiles have less of B, and short sums wait for
  // the other block at each tile: 512 -> 96 34, 34; 1 024 -> 64 52, 54; 2 048 -> 32 87, 89, and its dx, one slice, 75, 81; 8 bits, 384 -> 256
  // (three slices) 26, 27.
  const int pair_tiles = (int)(((int64_t)q.m + 2 * TILE_M - 1) / (2 * TILE_M));
  p->pair = !resident && nt >= 192 && nt % (b_mn ? 128 : 32) == 0 && p->KB >= 6 && (int64_t)pair_tiles * tiles_of(nt) * 2 >= sms;
  if (p->pair) {
    p->m_tiles = pair_tiles;
    p->b_slice = slice(nt / 2);
  }
  p->resident = resident;
  p->turns = (nt / PIECE + p->wide - 1) / p->wide;
  const int columns = resident ? nt : p->n_tiles * nt;
  p->lasting = columns <= LASTING ? columns : 0;
  p->tmem_cols = 32;
  while (p->tmem_cols < p->accs * nt) p->tmem_cols *= 2;
}

template <int KIND, bool B_MN, int ACT, bool GRAD, bool BF16, bool PAIR> int launch_as(Params& p, cudaStream_t st) {
  const wcn_linear_product& q = p.q;
  constexpr int size = KIND == WCN_E4M3 ? 1 : 2, depth = SLICE_BYTES / size;
  constexpr CUtensorMapDataType wide = BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  constexpr CUtensorMapDataType type = KIND == WCN_E4M3 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : wide;
  const int stage = p.resident ? A_BYTES : A_BYTES + p.b_slice, kept = p.resident ? p.KB * p.b_slice : 0;
  p.stages = (SMEM_BUDGET - FIXED - kept) / stage;
  if (p.stages > MAX_STAGES) p.stages = MAX_STAGES;
  if (p.stages < 2) return WCN_ERR_UNSUPPORTED_CONFIG;
  CUtensorMap a, b, out, add;
  EncodeTiledFn encode = encode_tiled();
  if (!encode) return WCN_ERR_UNSUPPORTED_CONFIG;
  bool ok = box_map(encode, &a, type, size, q.a, q.m, q.k, q.a_ld, depth, TILE_M);
  ok = ok && (B_MN ? box_map(encode, &b, type, size, q.b, q.k, q.n, q.b_ld, 64, 64) : box_map(encode, &b, type, size, q.b, q.n, q.k, q.b_ld, depth, PAIR ? p.NT / 2 : p.NT));
  out = add = a;   // (not used where they are not made)
  if (p.out_tma) ok = ok && box_map(encode, &out, wide, 2, q.out, q.m, q.n, q.out_ld, PIECE, 32);
  if (q.add && p.add_tma) ok = ok && box_map(encode, &add, wide, 2, q.add, q.m, q.n, q.add_ld, PIECE, 32);
  if (!ok) return WCN_ERR_UNSUPPORTED_CONFIG;
  constexpr auto kern = linear_kernel<KIND, B_MN, ACT, GRAD, BF16, PAIR>;
  if (!allow_smem<kern>()) return WCN_ERR_INITIALIZATION;
  const size_t smem = (size_t)FIXED + kept + (size_t)p.stages * stage;
  const int sms = wcn_num_sms();
  const int64_t tiles = (int64_t)p.m_tiles * p.n_tiles;
  ++wcn_launched;
  if (PAIR) return wcn_launch(kern, dim3((unsigned)(2 * (tiles < sms / 2 ? tiles : sms / 2))), dim3(THREADS), smem, st, 2, a, b, out, add, p);
  kern<<<(unsigned)(tiles < sms ? tiles : sms), THREADS, smem, st>>>(a, b, out, add, p);
  return cudaGetLastError() == cudaSuccess ? WCN_OK : WCN_ERR_EXECUTION;
}

template <int KIND, bool B_MN, int ACT, bool GRAD, bool BF16> int launch(const wcn_linear_product& q, int32_t* dev_status, cudaStream_t st) {
  Params p = {};
  p.q = q;
  p.dev_status = dev_status;
  p.out_tma = tma_rows(q.out, q.out_ld, 2);
  p.add_tma = q.add && tma_rows(q.add, q.add_ld, 2);
  p.wide = q.add ? 1 : 2;
  plan(q, KIND, B_MN, &p);
  return p.pair ? launch_as<KIND, B_MN, ACT, GRAD, BF16, true>(p, st) : launch_as<KIND, B_MN, ACT, GRAD, BF16, false>(p, st);
}

template <int KIND, bool GRAD, bool BF16> int by_act(const wcn_linear_product& q, int32_t* dev_status, cudaStream_t st) {
  switch (q.act) {
    case WCN_ACT_RELU: return launch<KIND, false, WCN_ACT_RELU, GRAD, BF16>(q, dev_status, st);
    case WCN_ACT_SILU: return launch<KIND, false, WCN_ACT_SILU, GRAD, BF16>(q, dev_status, st);
    case WCN_ACT_GELU: return launch<KIND, false, WCN_ACT_GELU, GRAD, BF16>(q, dev_status, st);
    default: return launch<KIND, false, WCN_ACT_NONE, GRAD, BF16>(q, dev_status, st);
  }
}

}  // namespace

// An activation, dropout or bias only with B as [n][k].  kind: WCN_F16, WCN_BF16 (the type of all) or WCN_E4M3 (of A and B; `bf16`: the others').  by_k: B is [k][n].  Rows of A and B start
// on 16-byte boundaries.
int wcn_linear_run(const wcn_linear_product& q, int kind, bool bf16, bool by_k, int32_t* dev_status, cudaStream_t st) {
  const int size = kind == WCN_E4M3 ? 1 : 2;
  if (!tma_rows(q.a, q.a_ld, size) || !tma_rows(q.b, q.b_ld, size)) return WCN_ERR_INVALID_PARAMETERS;
  if (kind == WCN_E4M3) return bf16 ? by_act<WCN_E4M3, false, true>(q, dev_status, st) : by_act<WCN_E4M3, false, false>(q, dev_status, st);
  if (by_k) return kind == WCN_BF16 ? launch<WCN_BF16, true, WCN_ACT_NONE, false, true>(q, dev_status, st) : launch<WCN_F16, true, WCN_ACT_NONE, false, false>(q, dev_status, st);
  if (q.grad) return kind == WCN_BF16 ? by_act<WCN_BF16, true, true>(q, dev_status, st) : by_act<WCN_F16, true, false>(q, dev_status, st);
  return kind == WCN_BF16 ? by_act<WCN_BF16, false, true>(q, dev_status, st) : by_act<WCN_F16, false, false>(q, dev_status, st);
}
