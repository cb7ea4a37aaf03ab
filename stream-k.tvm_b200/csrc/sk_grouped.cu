// Products grouped by expert with ragged sizes (sk_gemm_grouped): the rows of A are sorted by
// group, group e holding rows offsets[e] .. offsets[e+1), and every group has a matrix of its own.
//
//   NT   C[t,:] = B[e] A[t,:]            B [E,N,K]   (a linear layer of every expert)
//   NN   C[t,:] = A[t,:] B[e]            B [E,K,N]   (its input gradient)
//   TN   C[e]   = sum_t A[t,:]^T B[t,:]  C [E,K,N]   (its weight gradient)
//
// The sizes live on the device: every CTA reads the offsets, makes their prefix sums of tiles in
// shared memory, and walks its share of the tile list (a persistent launch, no host round trip).
// Offsets are clamped into [0, T] and made ascending before use, so no table of offsets makes a
// kernel read or write out of range; a table that needed it is reported through the status word.
//
// NT and NN: CTA pairs (cta_group::2).  The weights feed the UMMA M dimension (256 of the N output
// features per pair, 128 per CTA) and the rows of a group the UMMA N dimension, whose extent the
// instruction descriptor sets tile by tile in steps of 16: a group of 5 rows costs the tensor
// cores 32 columns and a group of 300 two tiles of 160 (150 rounded up), where rows on the M side
// would cost whole multiples of 128 or 256.  Groups of a few rows are then what they should be, a stream of the
// weights.  A pair's accumulator is transposed (lane = feature, column = row of A); a warp turns
// 32 x 32 of it through shared memory (ldmatrix.trans) and stores 64 contiguous bytes of a row of
// C with every four lanes.  (Stored straight from the registers, two bytes per lane, short sums paid
// for it: 9472 x 8192 x 512 89 us, turned 63.)
//
// What bounds them.  Few rows per group: the stream of the weights (16 rows over eight groups of
// 11008 x 4096: 112-115 us, 96-98 % of the rate of a copy).  Many rows: the tensor cores, 89 % of their
// cycles at 4 x 8192 x 4096 with 1000 rows each, and under a long load the power limit (16384 rows,
// 8 x 11008 x 4096: 0.97 ms, 1.52 PFLOP/s, alone; 1.13 ms among others like it).  In between: what an
// SM can load, 32 KB per step and CTA.
//
// TN: the sum runs over a group's rows, so both operands are MN-major (TMA boxes of 64 columns x
// 64 rows) and a group's last step holds rows of the next group.  Those must not count, whatever
// they hold: UMMAs past the group's end are not issued (16 rows each), and the rows of the last
// one that lie past it are zeroed in shared memory, in both operands (0 x NaN is NaN).  A last step
// of up to 16 or 32 rows loads only as many (60 groups of 5 rows, 1408 x 2048: 80 us with 64 loaded
// and zeroed piece by piece, 64 now).  Long sums are
// bound like the other two (16384 rows, 8 x 11008 x 4096: 0.98 ms), short ones by the writing of C
// (32 groups of 128 rows, 4096 x 2048 in fp32: 223 us, 4.8 TB/s; of 100 rows 202 us, 5.3; zeros alone 6.0).
#include "sk_common.cuh"
#include "sk_epilogue.cuh"

namespace {

using namespace skptx;

constexpr int BK = 64;                  // K per step: 128 bytes of a row
constexpr int HALF_M = 128;             // UMMA M rows per CTA of a pair
constexpr int A_STEP_BYTES = HALF_M * BK * 2;   // 16 KB
constexpr int MAX_BN = 256;
constexpr int MAX_STAGES = 12;
constexpr int EPI_WARPS = 8;
constexpr int TMEM_COLS = 512;
constexpr int SMEM_LIMIT = 232448;
constexpr int CTRL_BYTES = 512;

struct GroupedParams {
  int T, E, N, K;
  long long ldc, stride_c;   // elements
  const void* offsets;
  int off64;
  SkDiv d_rows[4];           // NT / NN: / tile_rows(bn_max, j)
  int bn_max;                // UMMA N of a tile: NT / NN: at most (rows of a group), a multiple of 32; TN: columns of N
  int tiles_f;               // tiles along the UMMA M side (NT / NN: of N; TN: of K)
  int steps;                 // NT / NN: K steps of a tile
  SkDiv d_steps;
  int tiles_n;               // TN: tiles of N
  int parts;                 // TN: pairs that may share a tile's sum
  int band;                  // TN: tiles of K that are walked side by side
  SkDiv d_band, d_in, d_last;   // / (band * tiles_n), / band, / the last band's tiles
  int stages;
  int b_step_bytes;          // shared memory per step of this CTA's half of the UMMA N operand
  int zero_rest;             // NT / NN: rows of C that belong to no group are set to zero
  int c_vec_ok, c_words;     // rows of C can take 16-byte stores; 4-byte stores
  int c_tma;                 // TN: C leaves through TMA stores
  int c_flat;                // TN: and every C[e] is one piece of memory
  int c_stream;              // TN: C is larger than L2, and leaves it first
  uint32_t idesc;            // with N = 0
  unsigned long long timeout_ns;
  SkWorkspace ws;
};

// NT / NN: how the tiles are dealt out (made on the device, the same in every CTA).  Tiles [0, sk)
// are Stream-K'd: their sk * steps steps go in equal contiguous runs to the first `runs` pairs, f
// each and one more for the first r; the rest go whole, one after the other, to all pairs.  (Only
// a launch of few tiles is split.  Splitting the last wave of a larger one was measured slower:
// few rows per group are bound by the stream of weights, whichever pairs draw it, and the parts of
// tiles of many rows are 128 KB per CTA each: 8 x 4096 x 4096, 4000 rows: 116 us against 109.)
struct RowPlan {
  int total, sk, runs, f, r;
};

struct Ctrl {
  uint64_t full[MAX_STAGES];        // leader: both CTAs' loads
  uint64_t empty[MAX_STAGES];       // each CTA
  uint64_t tail_full[MAX_STAGES];   // TN, each CTA: this CTA's loads of a stage that needs zeroing
  uint64_t tail_ready[MAX_STAGES];  // TN, leader: both CTAs' halves are zeroed
  uint64_t tmem_full[2], tmem_empty[2];
  uint32_t tmem_base;
  uint32_t abort;
  uint32_t last;                    // the epilogue's: this CTA was the last contributor to a split tile
  RowPlan plan;
};
static_assert(sizeof(Ctrl) <= CTRL_BYTES, "Ctrl must fit its reserved space");

constexpr int SK_MAX_PARTS = 4;   // most pairs that share a tile's sum

__host__ __device__ constexpr int align_up(int v, int a) { return (v + a - 1) / a * a; }
// Group table in shared memory: start[E + 1], then (NT / NN) first[E + 1], the first row tile, then
// what make_table passes between its warps, five numbers for every 32 of the E + 1.
__host__ __device__ constexpr int table_chunks(int E) { return (E + 32) / 32; }
__host__ __device__ constexpr int table_bytes(int E, bool tiles) {
  return align_up(((tiles ? 2 : 1) * (E + 1) + 5 * table_chunks(E)) * 4, 16);
}

// Rows per tile, choice j: bn_max, a half, a quarter, an eighth of it (multiples of 16, at least 32).
__host__ __device__ __forceinline__ int tile_rows(int bn_max, int j) {
  const int v = align_up(bn_max >> j, 16);
  return v < 32 ? 32 : v;
}

// Fills the table.  Called by every thread; ends with the table visible to all.  A warp takes 32
// of the E + 1 offsets at a time, and what passes from one 32 to the next (the running maximum of the
// starts, the numbers of tiles) goes through `scratch`: with hundreds of groups and a few rows the
// table is most of the launch (512 groups of 328 x 472, 10 rows: 31.2 us with one warp making it and
// every role looking for its tiles group by group, 8.3 now).
template <bool ROWS, bool SPLIT>
__device__ __forceinline__ void make_table(const GroupedParams& p, int* start, int* first, int* scratch, RowPlan* plan,
                                           int units) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int chunks = table_chunks(p.E);
  for (int c = warp; c < chunks; c += warps) {
    const int i = c * 32 + lane;
    int s = 0;
    if (i <= p.E) {
      long long o = p.off64 ? static_cast<const long long*>(p.offsets)[i]
                            : static_cast<long long>(static_cast<const int*>(p.offsets)[i]);
      bool bad = o < 0 || o > p.T;
      o = o < 0 ? 0 : o > p.T ? p.T : o;
      if (i > 0) {
        const long long before = p.off64 ? static_cast<const long long*>(p.offsets)[i - 1]
                                         : static_cast<long long>(static_cast<const int*>(p.offsets)[i - 1]);
        bad = bad || before > o;
      }
      s = static_cast<int>(o);
      if (bad && blockIdx.x == 0) sk_report(p.ws.status, SK_ERR_ARG, static_cast<uint32_t>(i), 0u);
    }
    __syncwarp();
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, s, d);
      if (lane >= d && o > s) s = o;
    }
    if (i <= p.E) start[i] = s;
    if (lane == 31) scratch[c] = s;
  }
  __syncthreads();
  for (int c = warp; c < chunks; c += warps) {
    const int i = c * 32 + lane;
    const int top = __reduce_max_sync(0xffffffffu, lane < c ? scratch[lane] : 0);   // (at most 33 chunks)
    int s = i <= p.E ? start[i] : 0;
    if (s < top) s = top;
    int before = __shfl_up_sync(0xffffffffu, s, 1);
    if (lane == 0) before = top;
    if (i <= p.E) start[i] = s;
#pragma unroll
    for (int j = 0; ROWS && j < 4; ++j) {   // tiles if a tile takes bn_max, bn_max / 2, / 4, / 8 rows
      const int n = i > 0 && i <= p.E ? sk_div(s - before + tile_rows(p.bn_max, j) - 1, p.d_rows[j]) : 0;
      const int all = __reduce_add_sync(0xffffffffu, n);
      if (lane == 0) scratch[(1 + j) * chunks + c] = all;
    }
  }
  __syncthreads();
  if constexpr (ROWS) {
    // Too few tiles for the pairs: fewer rows per tile, as long as every tile gets a pair of its
    // own (a step of 64 rows takes little more than half the time of one of 256).
    int bn = 0, total = 0;
    SkDiv d_bn = p.d_rows[0];
    const int* counts = scratch;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int* mine = scratch + (1 + j) * chunks;
      const int count = __reduce_add_sync(0xffffffffu, (lane < chunks ? mine[lane] : 0) + (lane == 0 && chunks > 32 ? mine[32] : 0));
      if (j == 0 || static_cast<long long>(count) * p.tiles_f <= units) {
        bn = tile_rows(p.bn_max, j);
        total = count * p.tiles_f;
        d_bn = p.d_rows[j];
        counts = mine;
      }
    }
    for (int c = warp; c < chunks; c += warps) {
      const int i = c * 32 + lane;
      const int earlier = __reduce_add_sync(0xffffffffu, lane < c ? counts[lane] : 0);
      // tiles of group i - 1; first[i] = tiles of groups 0 .. i - 1
      int t = i > 0 && i <= p.E ? sk_div(start[i] - start[i - 1] + bn - 1, d_bn) : 0;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, t, d);
        if (lane >= d) t += o;
      }
      if (i <= p.E) first[i] = earlier + t;
    }
    if (threadIdx.x == 0) {
      // Still no more tiles than half of the pairs, and long sums: split each over up to four
      // pairs, whose parts the last of them to finish adds (a part read back costs about 0.5 us
      // for 64 rows, so more pairs per tile would gain nothing).
      RowPlan q;
      q.total = total; q.sk = 0; q.runs = 1; q.f = 0; q.r = 0;
      if (SPLIT && total > 0 && 2 * total <= units) {
        q.sk = total;
        q.runs = units / total < SK_MAX_PARTS ? units / total * total : SK_MAX_PARTS * total;
        const int S = q.sk * p.steps;
        q.f = S / q.runs;
        q.r = S - q.f * q.runs;
      }
      *plan = q;
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------- NT and NN
struct RowTile {
  int tile, k0, k1;   // steps [k0, k1) of it
  int e;          // group
  int f0;         // first output feature of the pair's 256
  int r0, rows;   // rows of A
  int bn;         // UMMA N: rows rounded up to 16, at least 32
};

// First step of run p; the run that step i belongs to.
__device__ __forceinline__ int run_begin(const RowPlan& q, int p) {
  return p < q.runs ? p * q.f + (p < q.r ? p : q.r) : q.runs * q.f + q.r;
}
__device__ __forceinline__ int run_of(const RowPlan& q, int i) {
  const int big = q.r * (q.f + 1);
  return i < big ? i / (q.f + 1) : q.r + (i - big) / q.f;
}

// Walks a pair's run, then the whole tiles sk + unit, sk + unit + units, ...  The tiles are
// numbered group by group, inside a group in bands of up to eight row tiles, the feature tiles of
// a band one after the other (the pairs that run at a time then share few weight panels and few
// row panels).
struct RowWalk {
  int it, it_end, t, e;
  __device__ __forceinline__ void init(const RowPlan& q, int unit) {
    it = run_begin(q, unit);
    it_end = run_begin(q, unit + 1);
    t = q.sk + unit;
    e = 0;
  }
  __device__ __forceinline__ bool next(const GroupedParams& p, const RowPlan& q, const int* start, const int* first,
                                       int units, RowTile& o) {
    if (it < it_end) {
      o.tile = sk_div(it, p.d_steps);
      o.k0 = it - o.tile * p.steps;
      o.k1 = p.steps - o.k0 < it_end - it ? p.steps : o.k0 + (it_end - it);
      it += o.k1 - o.k0;
    } else {
      if (t >= q.total) return false;
      o.tile = t;
      o.k0 = 0;
      o.k1 = p.steps;
      t += units;
    }
    if (first[e + 1] * p.tiles_f <= o.tile) {   // (whole warps walk: 32 groups at a look)
      for (const int lane = threadIdx.x & 31;; e += 32) {
        if (e >= p.E) return false;               // (not reached: o.tile < first[E] * tiles_f)
        const int i = e + 1 + lane < p.E ? e + 1 + lane : p.E;
        const unsigned past = __ballot_sync(0xffffffffu, first[i] * p.tiles_f > o.tile);
        if (past != 0u) {
          e += __ffs(past) - 1;
          break;
        }
      }
    }
    const int mt = first[e + 1] - first[e];
    int local = o.tile - first[e] * p.tiles_f;
    const int band = local / (8 * p.tiles_f);
    local -= band * 8 * p.tiles_f;
    const int in_band = mt - band * 8 < 8 ? mt - band * 8 : 8;
    const int f = local / in_band;
    const int m = band * 8 + (local - f * in_band);
    const int rows = start[e + 1] - start[e];
    const int per = (rows + mt - 1) / mt;         // the group's rows in equal tiles
    o.e = e;
    o.f0 = f * (2 * HALF_M);
    o.r0 = start[e] + m * per;
    o.rows = rows - m * per < per ? rows - m * per : per;
    o.bn = o.rows > 16 ? (o.rows + 15) & ~15 : 32;
    return true;
  }
};

constexpr int NT_THREADS = 64 + 32 * EPI_WARPS;   // warp 0 producer, 1 MMA issuer, 2..9 epilogue
constexpr int TURN_BYTES = 2048;                  // an epilogue warp's 32 features x 32 rows of A, 16 bits each

// Where a warp keeps piece k (8 rows of A, 16 bytes) of feature f while it turns a block: two
// features to 128 bytes, the pieces permuted so that neither the lanes that write (eight
// consecutive features, one piece) nor the matrices read back (features 8 j + 2 m and + 1 for
// j = 0..3) meet on a bank.
__device__ __forceinline__ uint32_t turn_at(int f, int k) {
  const int swap = ((f >> 1) ^ (f >> 3)) & 3;
  return static_cast<uint32_t>((f >> 1) * 128 + ((f & 1) * 4 + (k ^ swap)) * 16);
}

// W_MN: the weights are MN-major (NN): two boxes of 64 features x 64 of K per step.  BF16: C's type.
// SPLIT: the launch may split tiles (a kernel without that code is ahead on small launches: every
// line of code it touches is an instruction-cache miss).
template <bool W_MN, bool BF16, bool SPLIT>
__global__ void __launch_bounds__(NT_THREADS, 1)
sk_grouped_rows_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX16,
                       const __grid_constant__ CUtensorMap tmX64, const __grid_constant__ CUtensorMap tmX128,
                       uint16_t* __restrict__ C, const GroupedParams p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t base = (raw_addr + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - raw_addr);
  const int STAGES = p.stages;
  const uint32_t sW = base, sX = base + STAGES * A_STEP_BYTES;
  Ctrl* ctrl = reinterpret_cast<Ctrl*>(smem + STAGES * (A_STEP_BYTES + p.b_step_bytes));
  int* start = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(ctrl) + CTRL_BYTES + EPI_WARPS * TURN_BYTES);
  int* first = start + p.E + 1;
  volatile uint32_t* abort_flag = &ctrl->abort;
  const int warp = uniform_warp_idx(), lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const int unit = blockIdx.x >> 1, units = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(smem_u32(&ctrl->full[i]), 1);
      mbar_init(smem_u32(&ctrl->empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&ctrl->tmem_full[i]), 1);
      mbar_init(smem_u32(&ctrl->tmem_empty[i]), 2 * EPI_WARPS);
    }
    ctrl->abort = 0u;
    fence_mbar_init();
    fence_proxy_async_smem();
    prefetch_tensormap(&tmW);
    prefetch_tensormap(&tmX16);
    if (p.bn_max > 32) prefetch_tensormap(&tmX64);
    if (p.bn_max > 128) prefetch_tensormap(&tmX128);
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(&ctrl->tmem_base), TMEM_COLS);
    tmem_relinquish_pair();
    if (lane == 0) griddep_launch_dependents();   // the next kernel of the stream may begin its own start-up
  }
  griddep_wait();
  make_table<true, SPLIT>(p, start, first, first + p.E + 1, &ctrl->plan, units);
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(&ctrl->tmem_base);
  const RowPlan plan = ctrl->plan;
  RowWalk walk;
  walk.init(plan, unit);
  RowTile tile;

  // (The single-thread roles are run by their whole warp, with the TMA, mbarrier and tcgen05
  // instructions behind an elected lane: warp-uniform code issues them at half the cost.)
  if (warp == 0) {
    // ------------------------------------------------------------- producer (both CTAs)
    {
      const bool leader = elect_one();
      int stage = 0;
      uint32_t ph = 0;
      bool ok = true;
      const uint32_t full0 = smem_u32(&ctrl->full[0]), empty0 = smem_u32(&ctrl->empty[0]);
      const uint32_t full0_leader = mapa_shared(full0, 0);
      while (ok && walk.next(p, plan, start, first, units, tile)) {
        const int half = tile.bn / 2;             // rows of A that this CTA supplies
        const CUtensorMap* tmX = half <= 16 ? &tmX16 : half <= 64 ? &tmX64 : &tmX128;
        const int box = half <= 16 ? 16 : half <= 64 ? 64 : 128;
        const uint32_t tx = 2u * (A_STEP_BYTES + static_cast<uint32_t>(box) * 128u);   // of both CTAs
        const int f_row = tile.f0 + rank * HALF_M, x_row = tile.r0 + rank * half;
        for (int k = tile.k0; k < tile.k1; ++k) {
          if (!sk_wait_bar_warp(empty0 + 8u * stage, ph ^ 1u, abort_flag, p, stage, 0)) {
            ok = false;
            break;
          }
          const uint32_t bar = full0_leader + 8u * stage;
          if (leader) {
            if (rank == 0) mbar_arrive_expect_tx(full0 + 8u * stage, tx);
            const uint32_t dW = sW + stage * A_STEP_BYTES;
            if constexpr (W_MN) {
              tma_load_3d_pair(dW, &tmW, bar, f_row, k * BK, tile.e);
              tma_load_3d_pair(dW + 8192, &tmW, bar, f_row + 64, k * BK, tile.e);
            } else {
              tma_load_3d_pair(dW, &tmW, bar, k * BK, f_row, tile.e);
            }
            tma_load_2d_pair(sX + stage * p.b_step_bytes, tmX, bar, k * BK, x_row);
          }
          if (++stage == STAGES) { stage = 0; ph ^= 1u; }
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------- MMA issuer (leader)
    if (rank == 0) {
      const bool leader = elect_one();
      int stage = 0;
      uint32_t ph = 0, nseg = 0;
      bool ok = true;
      constexpr uint32_t w_kstep16 = (W_MN ? 2048u : 32u) >> 4;
      const uint64_t w_hi = umma_desc_sw128_hi(W_MN ? 8192u : 16u, 1024), x_hi = umma_desc_sw128_hi(16u, 1024);
      const uint32_t w_lo0 = umma_desc_lo(sW), x_lo0 = umma_desc_lo(sX);
      const uint32_t full0 = smem_u32(&ctrl->full[0]), empty0 = smem_u32(&ctrl->empty[0]);
      while (ok && walk.next(p, plan, start, first, units, tile)) {
        const uint32_t buf = nseg & 1u;
        if (!sk_wait_bar_warp(smem_u32(&ctrl->tmem_empty[buf]), ((nseg >> 1) & 1u) ^ 1u, abort_flag, p, 16 + buf, 1)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + buf * MAX_BN;
        const uint32_t idesc = p.idesc | (static_cast<uint32_t>(tile.bn >> 3) << 17);
        uint32_t accumulate = 0u;
        for (int k = tile.k0; k < tile.k1; ++k) {
          if (!sk_wait_bar_warp(full0 + 8u * stage, ph, abort_flag, p, 32 + stage, 1)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t w_lo = w_lo0 + stage * (A_STEP_BYTES >> 4);
          const uint32_t x_lo = x_lo0 + stage * (static_cast<uint32_t>(p.b_step_bytes) >> 4);
#pragma unroll
          for (int kk = 0; kk < BK / 16; ++kk) {
            if (leader)
              umma_f16_ss_pair(d_tmem, w_hi | (w_lo + kk * w_kstep16), x_hi | (x_lo + kk * 2), idesc, accumulate);
            accumulate = 1u;
          }
          if (leader) umma_commit_pair(empty0 + 8u * stage);
          if (++stage == STAGES) { stage = 0; ph ^= 1u; }
        }
        if (!ok) break;
        if (leader) umma_commit_pair(smem_u32(&ctrl->tmem_full[buf]));
        ++nseg;
      }
    }
  } else {
    // ------------------------------------------------------------- epilogue (both CTAs)
    const int q = warp & 3, sub = (warp - 2) >> 2;   // TMEM lane quadrant; which of its two warps
    if (p.zero_rest) {
      // rows before the first group and after the last, while the first tile is on its way
      const int lo = start[0], hi = start[p.E], rest = lo + (p.T - hi);
      const int nw = gridDim.x * EPI_WARPS;
      for (int i = blockIdx.x * EPI_WARPS + (warp - 2); i < rest; i += nw) {
        uint16_t* row = C + static_cast<long long>(i < lo ? i : hi + (i - lo)) * p.ldc;
        if (p.c_vec_ok) {
          for (int c = lane * 8; c + 8 <= p.N; c += 256) *reinterpret_cast<uint4*>(row + c) = make_uint4(0u, 0u, 0u, 0u);
          for (int c = (p.N & ~7) + lane; c < p.N; c += 32) row[c] = 0;
        } else {
          for (int c = lane; c < p.N; c += 32) row[c] = 0;
        }
      }
    }
    const uint32_t tmem_full0 = smem_u32(&ctrl->tmem_full[0]);
    const uint32_t tmem_empty0 = mapa_shared(smem_u32(&ctrl->tmem_empty[0]), 0);
    const uint32_t turn = smem_u32(ctrl) + CTRL_BYTES + (warp - 2) * TURN_BYTES;
    const int turn_f = 8 * ((lane & 7) >> 1) + 2 * (lane >> 3) + (lane & 1);   // the feature whose piece this lane names
    uint32_t nseg = 0;
    bool dead = false;
    // Turned block -> C: this lane stores features f .. f + 7 of row `row` of C.
    auto store8 = [&](long long row, int f, const uint32_t (&w)[4]) {
      uint16_t* d = C + row * p.ldc + f;
      if (p.c_vec_ok && f + 8 <= p.N) {
        *reinterpret_cast<uint4*>(d) = make_uint4(w[0], w[1], w[2], w[3]);
      } else if (p.c_words && f + 8 <= p.N) {
#pragma unroll
        for (int i = 0; i < 4; ++i) reinterpret_cast<uint32_t*>(d)[i] = w[i];
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (f + i < p.N) d[i] = static_cast<uint16_t>(w[i >> 1] >> (16 * (i & 1)));
      }
    };
    // Eight columns (rows of A) of this lane's feature -> piece k of the warp's block.
    auto turn_in = [&](int k, const float (&v)[8]) {
      const uint32_t w0 = sk_pack2(v[0], v[1], BF16), w1 = sk_pack2(v[2], v[3], BF16);
      const uint32_t w2 = sk_pack2(v[4], v[5], BF16), w3 = sk_pack2(v[6], v[7], BF16);
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(turn + turn_at(lane, k)), "r"(w0), "r"(w1), "r"(w2),
                   "r"(w3)
                   : "memory");
    };
    while (walk.next(p, plan, start, first, units, tile)) {
      const uint32_t buf = nseg & 1u;
      if (!dead) {
        const bool got = sk_wait_bar(tmem_full0 + 8u * buf, (nseg >> 1) & 1u, abort_flag, p, 24 + buf, 2);
        if (!__all_sync(0xffffffffu, got)) dead = true;
      }
      ++nseg;
      tc_fence_after();
      const uint32_t t_addr = tmem_base + buf * MAX_BN + (static_cast<uint32_t>(q * 32) << 16);
      const int fc = tile.f0 + rank * HALF_M;               // the CTA's 128 features
      const bool whole = !SPLIT || (tile.k0 == 0 && tile.k1 == p.steps);
      const int me = unit * 2 + rank;
      float* const mine = p.ws.part_slots + static_cast<size_t>(2 * me + (tile.k0 == 0 ? 1 : 0)) * SK_SLOT_FLOATS;
      if (!dead && fc + q * 32 < p.N) {
        for (int c = sub * 32; c < tile.rows; c += 64) {
          uint32_t v[32];
          tmem_ld_32x32(t_addr + c, v);
          tmem_ld_wait();
          if (whole) {
            __syncwarp();                                   // the block before has been read
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              float x[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(v[8 * k + i]);
              turn_in(k, x);
            }
            __syncwarp();
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              uint32_t w[4];
              ldmatrix_x4_trans(turn + turn_at(turn_f, k), w);
              const int row = c + 8 * k + (lane >> 2);
              if (row < tile.rows) store8(tile.r0 + row, fc + q * 32 + 8 * (lane & 3), w);
            }
          } else {
            // a part of the sum: fp32, four columns of a feature together (a warp: 512 bytes)
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (c + 4 * j < tile.rows)
                __stcg(reinterpret_cast<uint4*>(mine) + (c / 4 + j) * HALF_M + q * 32 + lane,
                       make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]));
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster_relaxed(tmem_empty0 + 8u * buf);
      if (whole) continue;

      // A split tile: whoever arrives last adds the parts, in the order of K, and stores.  Nobody
      // waits for anyone, so the kernel needs no two CTAs to run at the same time.
      const int c_first = run_of(plan, tile.tile * p.steps), c_last = run_of(plan, tile.tile * p.steps + p.steps - 1);
      __threadfence();
      named_bar_sync(SK_EPI_BAR_ID, 32 * EPI_WARPS);
      if (threadIdx.x == 64) {
        uint32_t* const count = p.ws.counters + c_first * 2 + rank;
        const uint32_t old = atom_add_acqrel_u32(count, 1u);
        const bool last = old == static_cast<uint32_t>(c_last - c_first);
        if (last) *count = 0u;                              // zero between launches
        *reinterpret_cast<volatile uint32_t*>(&ctrl->last) = last ? 1u : 0u;
      }
      named_bar_sync(SK_EPI_BAR_ID, 32 * EPI_WARPS);
      const bool last = *reinterpret_cast<volatile uint32_t*>(&ctrl->last) != 0u;
      named_bar_sync(SK_EPI_BAR_ID, 32 * EPI_WARPS);        // (read before the next tile's is written)
      if (!last) continue;
      __threadfence();
      const int pieces = (tile.rows + 7) >> 3;
      for (int i = warp - 2; i < 4 * pieces; i += EPI_WARPS) {
        const int qq = i & 3, piece = i >> 2;
        if (fc + qq * 32 >= p.N) continue;
        const size_t at = static_cast<size_t>(piece * 2) * HALF_M + qq * 32 + lane;
        // (columns past the tile's rows hold anything; their rows of C are not stored)
        const bool second = piece * 8 + 4 < tile.rows;
        float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        for (int u0 = c_first; u0 <= c_last; u0 += 4) {
          float4 x[4][2];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int u = u0 + j <= c_last ? u0 + j : c_last;   // (a repeated fetch, not added)
            const float4* src = reinterpret_cast<const float4*>(
                                    p.ws.part_slots + static_cast<size_t>(2 * (u * 2 + rank) + (u == c_first ? 1 : 0)) * SK_SLOT_FLOATS) + at;
            x[j][0] = __ldcg(src);
            x[j][1] = second ? __ldcg(src + HALF_M) : make_float4(0.f, 0.f, 0.f, 0.f);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (u0 + j <= c_last) {
              acc[0] += x[j][0].x; acc[1] += x[j][0].y; acc[2] += x[j][0].z; acc[3] += x[j][0].w;
              acc[4] += x[j][1].x; acc[5] += x[j][1].y; acc[6] += x[j][1].z; acc[7] += x[j][1].w;
            }
        }
        __syncwarp();
        turn_in(0, acc);
        __syncwarp();
        uint32_t w[4];
        ldmatrix_x4_trans(turn + turn_at(turn_f, 0), w);
        const int row = piece * 8 + (lane >> 2);
        if (row < tile.rows) store8(tile.r0 + row, fc + qq * 32 + 8 * (lane & 3), w);
      }
    }
  }

  // ------------------------------------------------------------- teardown
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  if (warp == 1) {
    if (*abort_flag) {
      const unsigned long long t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 200000ULL) __nanosleep(1000);
    }
    tc_fence_after();
    __syncwarp();
    tmem_dealloc_pair(tmem_base, TMEM_COLS);
  }
}

// ------------------------------------------------------------------------------- TN
struct SumTile {
  int e, f0, c0;    // group, first row (of K) and column (of N) of the pair's 256 x 256 tile of C[e]
  int r0, rows;     // the group's rows of A and B
  int local;        // number of the tile inside its group
  int k0, k1;       // steps of 64 rows to add up: all of them, or part `part` of `parts`
  int part, parts;
};

// Walks the items unit, unit + units, ...; an item is a tile, or with p.parts > 1 (as many items as
// pairs or fewer) one of the parts of a tile's sum.  A group with fewer than SUM_MIN_RUN steps for
// every part has fewer of them; the rest of its items are skipped.
constexpr int SUM_MIN_RUN = 16;
template <bool SPLIT>
struct SumWalk {
  int t, e, part;   // tile of group e (it may still lie in a later group)
  __device__ __forceinline__ void init(const GroupedParams& p, int unit) {
    t = SPLIT ? unit / p.parts : unit;
    part = SPLIT ? unit - t * p.parts : 0;
    e = 0;
  }
  __device__ __forceinline__ bool next(const GroupedParams& p, const int* start, int units, SumTile& o) {
    const int per_e = p.tiles_f * p.tiles_n;
    while (t >= per_e && e < p.E) { t -= per_e; ++e; }
    if (e >= p.E) return false;
    const int steps = (start[e + 1] - start[e] + BK - 1) / BK;
    o.local = t;
    o.k0 = 0; o.k1 = steps; o.part = 0; o.parts = 1;
    if (SPLIT) {
      const int most = steps / SUM_MIN_RUN;
      o.parts = most < 1 ? 1 : most < p.parts ? most : p.parts;
      if (part >= o.parts) return false;
      o.part = part;
      o.k0 = static_cast<int>(static_cast<long long>(steps) * part / o.parts);
      o.k1 = static_cast<int>(static_cast<long long>(steps) * (part + 1) / o.parts);
    }
    const int band = sk_div(t, p.d_band);
    const int local = t - band * p.band * p.tiles_n;
    const int left = p.tiles_f - band * p.band;
    const int n = sk_div(local, left < p.band ? p.d_last : p.d_in);
    o.e = e;
    o.f0 = (band * p.band + (local - n * (left < p.band ? left : p.band))) * (2 * HALF_M);
    o.c0 = n * p.bn_max;
    o.r0 = start[e];
    o.rows = start[e + 1] - start[e];
    t += SPLIT ? p.E * per_e : units;   // (parts: one item per pair)
    return true;
  }
};

constexpr int TN_THREADS = NT_THREADS + 32;   // one warp more: it zeroes what lies past a group's end
constexpr int TN_B_STEP = 128 * BK * 2;
constexpr int TN_STEP = A_STEP_BYTES + TN_B_STEP;   // a stage holds one step

// Does step k of a group of `rows` rows hold a UMMA that reaches past the group's end?
__device__ __forceinline__ bool step_needs_zeros(int k, int rows) {
  return (k + 1) * BK > rows && (rows & 15) != 0;
}

// Tensor maps of A and B with boxes of 16, 32 and 64 rows.
struct alignas(64) SumMaps {
  CUtensorMap a[3], b[3];
};

constexpr int OUT_F16 = 0, OUT_BF16 = 1, OUT_F32 = 2;   // type of C

// LONG: a group may have more than SUM_RUN steps, and C is fp32.  The tensor cores' adders truncate: a sum
// that stays in tensor memory loses half a unit in the last place with every 16 rows, always towards
// zero, and with it the last bits that fp32 is asked for (8192 rows of normal numbers: off by 9.1e-6 in
// the norm).  So they add up SUM_RUN steps, 512 rows, at a time, and the epilogue adds those sums in
// registers, rounding to nearest: off by 4.8e-7 whatever the length.  It costs long sums 1-4 % (8 groups
// of 2048 rows, 11008 x 4096: 1205 -> 1245 us; of 500 rows, 4096 x 4096, one run: 153 and 155); runs of
// four steps are off by 2.4e-7 and cost 6 %.  (16-bit results are rounded a hundred times as coarsely.)
constexpr int SUM_RUN = 8;

template <int OUT, bool SPLIT, bool LONG>
__global__ void __launch_bounds__(TN_THREADS, 1)
sk_grouped_sum_kernel(const __grid_constant__ SumMaps maps, const __grid_constant__ CUtensorMap tmC,
                      void* __restrict__ Cv, const GroupedParams p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t base = (raw_addr + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - raw_addr);
  const int STAGES = p.stages;
  const uint32_t sA = base, sB = base + STAGES * A_STEP_BYTES;
  const uint32_t cstage = base + STAGES * TN_STEP;           // 8 x 4 KB staging of the TMA stores
  Ctrl* ctrl = reinterpret_cast<Ctrl*>(smem + STAGES * TN_STEP + EPI_WARPS * 4096);
  int* start = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(ctrl) + CTRL_BYTES);
  volatile uint32_t* abort_flag = &ctrl->abort;
  const int warp = uniform_warp_idx(), lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const int unit = blockIdx.x >> 1, units = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(smem_u32(&ctrl->full[i]), 1);
      mbar_init(smem_u32(&ctrl->empty[i]), 1);
      mbar_init(smem_u32(&ctrl->tail_full[i]), 1);
      mbar_init(smem_u32(&ctrl->tail_ready[i]), 2);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&ctrl->tmem_full[i]), 1);
      mbar_init(smem_u32(&ctrl->tmem_empty[i]), 2 * EPI_WARPS);
    }
    ctrl->abort = 0u;
    fence_mbar_init();
    fence_proxy_async_smem();
    for (int i = 0; i < 3; ++i) {
      prefetch_tensormap(&maps.a[i]);
      prefetch_tensormap(&maps.b[i]);
    }
    if (p.c_tma) prefetch_tensormap(&tmC);
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(&ctrl->tmem_base), TMEM_COLS);
    tmem_relinquish_pair();
    if (lane == 0) griddep_launch_dependents();   // the next kernel of the stream may begin its own start-up
  }
  griddep_wait();
  make_table<false, false>(p, start, nullptr, start + p.E + 1, nullptr, units);
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(&ctrl->tmem_base);
  SumWalk<SPLIT> walk;
  walk.init(p, unit);
  SumTile tile;

  if (warp == 0) {
    // ------------------------------------------------------------- producer (both CTAs)
    {
      const bool leader = elect_one();
      int stage = 0;
      uint32_t ph = 0;
      bool ok = true;
      const uint32_t full0 = smem_u32(&ctrl->full[0]), empty0 = smem_u32(&ctrl->empty[0]);
      const uint32_t tail0 = smem_u32(&ctrl->tail_full[0]);
      const uint32_t full0_leader = mapa_shared(full0, 0);
      while (ok && walk.next(p, start, units, tile)) {
        const int a_col = tile.f0 + rank * HALF_M, b_col = tile.c0 + rank * (p.bn_max / 2);
        for (int k = tile.k0; k < tile.k1; ++k) {
          if (!sk_wait_bar_warp(empty0 + 8u * stage, ph ^ 1u, abort_flag, p, stage, 0)) {
            ok = false;
            break;
          }
          // A stage that needs zeroing is announced in each CTA by itself: the zeroing warp has
          // to see its own CTA's bytes land.  (The leader's barrier completes a phase all the
          // same, so that the parities of the ring stay in step.)
          const bool tail = step_needs_zeros(k, tile.rows);
          const int b_chunks = p.bn_max / 128;            // of 64 columns
          // (a short step loads 16 or 32 rows: what lies past them no UMMA reads)
          const int left = tile.rows - k * BK, size = left <= 16 ? 0 : left <= 32 ? 1 : 2;
          const CUtensorMap *tmA = &maps.a[size], *tmB = &maps.b[size];
          const uint32_t bytes = (2 + b_chunks) * (2048u << size);
          uint32_t bar = full0_leader + 8u * stage;
          if (tail) bar = tail0 + 8u * stage;
          if (leader) {
            if (tail) {
              if (rank == 0) mbar_arrive(full0 + 8u * stage);
              mbar_arrive_expect_tx(bar, bytes);
            } else if (rank == 0) {
              mbar_arrive_expect_tx(full0 + 8u * stage, 2 * bytes);
            }
          }
          const uint32_t dA = sA + stage * A_STEP_BYTES, dB = sB + stage * TN_B_STEP;
          const int row = tile.r0 + k * BK;
          for (int h = 0; leader && h < 2; ++h) {
            if (tail) {
              tma_load_2d(dA + h * 8192, tmA, bar, a_col + h * 64, row);
              if (h < b_chunks) tma_load_2d(dB + h * 8192, tmB, bar, b_col + h * 64, row);
            } else {
              tma_load_2d_pair(dA + h * 8192, tmA, bar, a_col + h * 64, row);
              if (h < b_chunks) tma_load_2d_pair(dB + h * 8192, tmB, bar, b_col + h * 64, row);
            }
          }
          if (++stage == STAGES) { stage = 0; ph ^= 1u; }
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------- MMA issuer (leader)
    if (rank == 0) {
      const bool leader = elect_one();
      int stage = 0;
      uint32_t ph = 0, nseg = 0, tail_ph = 0;
      bool ok = true;
      const uint64_t hi = umma_desc_sw128_hi(8192u, 1024);   // MN-major: 64-wide chunks 8 KB apart, 8 rows 1 KB apart
      const uint32_t a_lo0 = umma_desc_lo(sA), b_lo0 = umma_desc_lo(sB);
      const uint32_t full0 = smem_u32(&ctrl->full[0]), empty0 = smem_u32(&ctrl->empty[0]);
      const uint32_t ready0 = smem_u32(&ctrl->tail_ready[0]);
      const uint32_t idesc = p.idesc | (static_cast<uint32_t>(p.bn_max >> 3) << 17);
      while (ok && walk.next(p, start, units, tile)) {
        if (tile.rows == 0) continue;   // (the epilogue writes zeros)
        for (int k = tile.k0; ok && k < tile.k1;) {
          const int run_end = LONG && tile.k1 - k > SUM_RUN ? k + SUM_RUN : tile.k1;
          const uint32_t buf = nseg & 1u;
          if (!sk_wait_bar_warp(smem_u32(&ctrl->tmem_empty[buf]), ((nseg >> 1) & 1u) ^ 1u, abort_flag, p, 16 + buf, 1)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t d_tmem = tmem_base + buf * MAX_BN;
          uint32_t accumulate = 0u;
          for (; k < run_end; ++k) {
            if (!sk_wait_bar_warp(full0 + 8u * stage, ph, abort_flag, p, 32 + stage, 1)) {
              ok = false;
              break;
            }
            if (step_needs_zeros(k, tile.rows)) {
              if (!sk_wait_bar_warp<true>(ready0 + 8u * stage, (tail_ph >> stage) & 1u, abort_flag, p, 48 + stage, 1)) {
                ok = false;
                break;
              }
              tail_ph ^= 1u << stage;
            }
            tc_fence_after();
            const uint32_t a_lo = a_lo0 + stage * (A_STEP_BYTES >> 4), b_lo = b_lo0 + stage * (TN_B_STEP >> 4);
            const int left = tile.rows - k * BK;              // rows of the group in this step
#pragma unroll
            for (int kk = 0; kk < BK / 16; ++kk) {
              if (leader && kk * 16 < left)
                umma_f16_ss_pair(d_tmem, hi | (a_lo + kk * 128), hi | (b_lo + kk * 128), idesc, accumulate);
              accumulate = 1u;
            }
            if (leader) umma_commit_pair(empty0 + 8u * stage);
            if (++stage == STAGES) { stage = 0; ph ^= 1u; }
          }
          if (!ok) break;
          if (leader) umma_commit_pair(smem_u32(&ctrl->tmem_full[buf]));
          ++nseg;
        }
      }
    }
  } else if (warp == 2 + EPI_WARPS) {
    // ------------------------------------------------------------- zeroing warp (both CTAs)
    int stage = 0;
    uint32_t tail_ph = 0;
    bool ok = true;
    const uint32_t tail0 = smem_u32(&ctrl->tail_full[0]);
    const uint32_t ready0_leader = mapa_shared(smem_u32(&ctrl->tail_ready[0]), 0);
    while (ok && walk.next(p, start, units, tile)) {
      for (int k = tile.k0; k < tile.k1; ++k) {
        if (step_needs_zeros(k, tile.rows)) {
          const bool got = sk_wait_bar(tail0 + 8u * stage, (tail_ph >> stage) & 1u, abort_flag, p, 56 + stage, 5);
          if (!__all_sync(0xffffffffu, got)) {
            ok = false;
            break;
          }
          tail_ph ^= 1u << stage;
          // rows lo .. hi of the step's 64, 128 bytes in each of the four chunks (swizzling moves
          // 16-byte pieces inside a row, so a whole row is a whole row)
          const int lo = tile.rows - k * BK, hi = (lo + 15) & ~15;
          const uint32_t a = sA + stage * A_STEP_BYTES, b = sB + stage * TN_B_STEP;
          for (int i = lo * 128 + lane * 16; i < hi * 128; i += 512) {
            st_shared_v4(a + i, 0.f, 0.f, 0.f, 0.f);
            st_shared_v4(a + 8192 + i, 0.f, 0.f, 0.f, 0.f);
            st_shared_v4(b + i, 0.f, 0.f, 0.f, 0.f);
            st_shared_v4(b + 8192 + i, 0.f, 0.f, 0.f, 0.f);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(ready0_leader + 8u * stage);
        }
        if (++stage == STAGES) stage = 0;
      }
    }
  } else {
    // ------------------------------------------------------------- epilogue (both CTAs)
    const int q = warp & 3, sub = (warp - 2) >> 2;
    const uint32_t tmem_full0 = smem_u32(&ctrl->tmem_full[0]);
    const uint32_t tmem_empty0 = mapa_shared(smem_u32(&ctrl->tmem_empty[0]), 0);
    const uint32_t buf_smem = cstage + static_cast<uint32_t>(warp - 2) * 4096u;
    constexpr bool F32 = OUT == OUT_F32;
    constexpr int gcols = F32 ? 32 : 64;            // columns of a 128-byte row of the staging buffer
    // 32 rows of gcols columns, this lane's row in v, to columns c.. of the tile: staged as 32 x 128
    // bytes, then one TMA store, or, where C's rows are not what TMA can address, a row at a time
    // with consecutive lanes on consecutive columns.
    auto store_group = [&](const SumTile& tile, int r0, int c, int valid, const float (&v)[gcols / 32][32]) {
      if (lane == 0) tma_store_wait_read<0>();
      __syncwarp();
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t a = buf_smem + static_cast<uint32_t>(lane) * 128u +
                           ((static_cast<uint32_t>(j) ^ (static_cast<uint32_t>(lane) & 7u)) << 4);
        if constexpr (F32) {
          st_shared_v4(a, v[0][4 * j], v[0][4 * j + 1], v[0][4 * j + 2], v[0][4 * j + 3]);
        } else {
          const float* w = &v[j >> 2][(j & 3) * 8];
          constexpr int BF = OUT == OUT_BF16;
          const uint32_t h0 = sk_pack2(w[0], w[1], BF), h1 = sk_pack2(w[2], w[3], BF);
          const uint32_t h2 = sk_pack2(w[4], w[5], BF), h3 = sk_pack2(w[6], w[7], BF);
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(h0), "r"(h1), "r"(h2), "r"(h3)
                       : "memory");
        }
      }
      // (TMA clips at the edges of C[e], but columns to whole 16 bytes: where N ends between, the rest of
      // them would be overwritten, so that group is stored by rows)
      if (p.c_tma && (valid - c >= gcols || ((valid - c) * (F32 ? 4 : 2) & 15) == 0)) {
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          if (p.c_stream) tma_store_3d_evict_first(&tmC, buf_smem, tile.c0 + c, r0, tile.e);
          else tma_store_3d(&tmC, buf_smem, tile.c0 + c, r0, tile.e);
          tma_store_commit();
        }
        return;
      }
      __syncwarp();
      const long long at = tile.e * p.stride_c + static_cast<long long>(r0) * p.ldc + tile.c0 + c;
      const int rows = p.K - r0 < 32 ? p.K - r0 : 32;
#pragma unroll 4
      for (int r = 0; r < rows; ++r) {
        const uint32_t row = buf_smem + r * 128;
        if constexpr (F32) {
          float w;
          asm volatile("ld.shared.f32 %0, [%1];"
                       : "=f"(w) : "r"(row + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4) : "memory");
          if (c + lane < valid) static_cast<float*>(Cv)[at + r * p.ldc + lane] = w;
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int i = h * 32 + lane;
            uint16_t w;
            asm volatile("ld.shared.u16 %0, [%1];"
                         : "=h"(w) : "r"(row + (((i >> 3) ^ (r & 7)) << 4) + (i & 7) * 2) : "memory");
            if (c + i < valid) static_cast<uint16_t*>(Cv)[at + r * p.ldc + i] = w;
          }
        }
      }
    };
    uint32_t nseg = 0;
    bool dead = false;
    while (walk.next(p, start, units, tile)) {
      const bool some = tile.rows > 0;
      if (!some && p.c_flat) {
        // an empty group whose matrix is one piece of memory: its tiles zero equal contiguous
        // shares of it, half a share per CTA
        const long long quads = static_cast<long long>(p.K) * p.N * (F32 ? 4 : 2) / 16;
        const long long tiles2 = 2LL * p.tiles_f * p.tiles_n, me = 2 * tile.local + rank;
        float4* base = reinterpret_cast<float4*>(static_cast<uint8_t*>(Cv) + tile.e * p.stride_c * (F32 ? 4 : 2));
        const long long end = quads * (me + 1) / tiles2;
        for (long long i = quads * me / tiles2 + (threadIdx.x - 64); i < end; i += 32 * EPI_WARPS)
          base[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        continue;
      }
      uint32_t buf = 0u;
      auto next_sum = [&]() {   // waits for the next accumulator
        buf = nseg & 1u;
        if (!dead) {
          const bool got = sk_wait_bar(tmem_full0 + 8u * buf, (nseg >> 1) & 1u, abort_flag, p, 24 + buf, 2);
          if (!__all_sync(0xffffffffu, got)) dead = true;
        }
        ++nseg;
        tc_fence_after();
        return tmem_base + buf * MAX_BN + (static_cast<uint32_t>(q * 32) << 16);
      };
      auto hand_back = [&]() {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster_relaxed(tmem_empty0 + 8u * buf);
      };
      const int r0 = tile.f0 + rank * HALF_M + q * 32;      // first of this warp's 32 rows of C[e]
      int valid = p.N - tile.c0;
      if (valid > p.bn_max) valid = p.bn_max;
      const bool whole = !SPLIT || tile.parts == 1;
      float4* const mine = reinterpret_cast<float4*>(p.ws.part_slots + static_cast<size_t>(2 * (unit * 2 + rank)) * SK_SLOT_FLOATS);
      bool one_run = true;
      if constexpr (LONG) {
        static_assert(F32, "16-bit results are rounded far above this");
        one_run = tile.k1 - tile.k0 <= SUM_RUN;
        if (!one_run) {
          float sum[MAX_BN / 64][1][32];
#pragma unroll
          for (int g = 0; g < MAX_BN / 64; ++g)
#pragma unroll
            for (int j = 0; j < 32; ++j) sum[g][0][j] = 0.f;
          for (int k = tile.k0; k < tile.k1; k += SUM_RUN) {
            const uint32_t t_addr = next_sum();
            if (!dead && r0 < p.K) {
#pragma unroll
              for (int g = 0; g < MAX_BN / 64; ++g) {
                const int c = (2 * g + sub) * 32;
                if (c < valid) {
#pragma unroll
                  for (int h = 0; h < 32; h += 16) {           // (sixteen at a time: registers)
                    uint32_t raw[16];
                    tmem_ld_32x16(t_addr + c + h, raw);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 16; ++j) sum[g][0][h + j] += __uint_as_float(raw[j]);
                  }
                }
              }
            }
            hand_back();
          }
          if (!dead && r0 < p.K) {
#pragma unroll
            for (int g = 0; g < MAX_BN / 64; ++g) {
              const int c = (2 * g + sub) * 32;
              if (c >= valid) break;
              if (whole) {
                store_group(tile, r0, c, valid, sum[g]);
              } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                  __stcg(mine + (c / 4 + j) * HALF_M + q * 32 + lane,
                         make_float4(sum[g][0][4 * j], sum[g][0][4 * j + 1], sum[g][0][4 * j + 2], sum[g][0][4 * j + 3]));
              }
            }
          }
        }
      }
      if (one_run) {
        const uint32_t t_addr = some ? next_sum() : 0u;
        if (!dead && r0 < p.K) {
          for (int c = sub * gcols; c < valid; c += 2 * gcols) {
            float v[gcols / 32][32];
            if (some) {
              uint32_t raw[gcols / 32][32];
#pragma unroll
              for (int h = 0; h < gcols / 32; ++h) tmem_ld_32x32(t_addr + c + h * 32, raw[h]);
              tmem_ld_wait();
#pragma unroll
              for (int h = 0; h < gcols / 32; ++h)
#pragma unroll
                for (int j = 0; j < 32; ++j) v[h][j] = __uint_as_float(raw[h][j]);
            } else {
#pragma unroll
              for (int h = 0; h < gcols / 32; ++h)
#pragma unroll
                for (int j = 0; j < 32; ++j) v[h][j] = 0.f;
            }
            if (whole) {
              store_group(tile, r0, c, valid, v);
            } else {
#pragma unroll
              for (int h = 0; h < gcols / 32; ++h)
#pragma unroll
                for (int j = 0; j < 8; ++j)
                  __stcg(mine + ((c + h * 32) / 4 + j) * HALF_M + q * 32 + lane,
                         make_float4(v[h][4 * j], v[h][4 * j + 1], v[h][4 * j + 2], v[h][4 * j + 3]));
            }
          }
        }
        if (some) hand_back();
      }
      if (whole) continue;

      // A sum in parts: the pairs unit - part .. unit - part + parts - 1 hold them; the last to arrive
      // adds them in order and stores (nobody waits for anyone).
      const int u0 = unit - tile.part;
      __threadfence();
      named_bar_sync(SK_EPI_BAR_ID, 32 * EPI_WARPS);
      if (threadIdx.x == 64) {
        uint32_t* const count = p.ws.counters + u0 * 2 + rank;
        const uint32_t old = atom_add_acqrel_u32(count, 1u);
        const bool last = old == static_cast<uint32_t>(tile.parts - 1);
        if (last) *count = 0u;                              // zero between launches
        *reinterpret_cast<volatile uint32_t*>(&ctrl->last) = last ? 1u : 0u;
      }
      named_bar_sync(SK_EPI_BAR_ID, 32 * EPI_WARPS);
      if (*reinterpret_cast<volatile uint32_t*>(&ctrl->last) == 0u) continue;   // (a pair has one item: no reuse)
      __threadfence();
      if (r0 < p.K) {
        for (int c = sub * gcols; c < valid; c += 2 * gcols) {
          float v[gcols / 32][32];
#pragma unroll
          for (int h = 0; h < gcols / 32; ++h)
#pragma unroll
            for (int j = 0; j < 32; ++j) v[h][j] = 0.f;
          const float4* src = reinterpret_cast<const float4*>(
                                  p.ws.part_slots + static_cast<size_t>(2 * (u0 * 2 + rank)) * SK_SLOT_FLOATS) +
                              (c / 4) * HALF_M + q * 32 + lane;
          constexpr size_t NEXT = SK_SLOT_FLOATS;          // float4s between the slots of two neighbouring pairs
#pragma unroll
          for (int h = 0; h < gcols / 32; ++h) {
            for (int u = 0; u < tile.parts; u += 2) {       // sixteen loads in flight, added in order
              float4 x[2][8];
#pragma unroll
              for (int j = 0; j < 8; ++j) x[0][j] = __ldcg(src + u * NEXT + (h * 8 + j) * HALF_M);
              const bool two = u + 1 < tile.parts;
#pragma unroll
              for (int j = 0; j < 8; ++j) x[1][j] = __ldcg(src + (two ? u + 1 : u) * NEXT + (h * 8 + j) * HALF_M);
#pragma unroll
              for (int w = 0; w < 2; ++w)
                if (w == 0 || two)
#pragma unroll
                  for (int j = 0; j < 8; ++j) {
                    v[h][4 * j] += x[w][j].x; v[h][4 * j + 1] += x[w][j].y;
                    v[h][4 * j + 2] += x[w][j].z; v[h][4 * j + 3] += x[w][j].w;
                  }
            }
          }
          store_group(tile, r0, c, valid, v);
        }
      }
    }
    if (lane == 0) tma_store_wait_read<0>();
  }

  // ------------------------------------------------------------- teardown
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  if (warp == 1) {
    if (*abort_flag) {
      const unsigned long long t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 200000ULL) __nanosleep(1000);
    }
    tc_fence_after();
    __syncwarp();
    tmem_dealloc_pair(tmem_base, TMEM_COLS);
  }
}

// ---------------------------------------------------------------- host side
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// [batch, rows, cols] tensor map (batch 0: two-dimensional), 128-byte swizzle, box {box_cols, box_rows(, 1)}.
int make_map(CUtensorMap* out, const void* ptr, bool f32, uint64_t batch, uint64_t rows, uint64_t cols, uint64_t ld,
             uint64_t batch_stride, uint32_t box_cols, uint32_t box_rows) {
  static EncodeTiledFn enc = []() -> EncodeTiledFn {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess) return nullptr;
    return q == cudaDriverEntryPointSuccess ? reinterpret_cast<EncodeTiledFn>(f) : nullptr;
  }();
  if (!enc) return SK_ERR_LAUNCH;
  const uint64_t esz = f32 ? 4 : 2;
  cuuint64_t gdim[3] = {cols, rows, batch};
  cuuint64_t gstride[2] = {ld * esz, batch_stride * esz};
  cuuint32_t box[3] = {box_cols, box_rows, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = enc(out, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, batch ? 3 : 2,
                         const_cast<void*>(ptr), gdim, gstride, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? SK_OK : sk_set_driver_error(static_cast<int>(r));
}

bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

}  // namespace

extern "C" int sk_gemm_grouped(const sk_grouped_problem* g, const void* A, const void* B, const void* offsets, void* C,
                               void* ws, size_t ws_bytes, void* stream) {
  if (!g || !A || !B || !C || !offsets) return SK_ERR_ARG;
  if (g->kind < SK_GROUPED_NT || g->kind > SK_GROUPED_TN) return SK_ERR_ARG;
  if (g->T <= 0 || g->E <= 0 || g->N <= 0 || g->K <= 0) return SK_ERR_SHAPE;
  if (g->E > SK_GROUPED_MAX_GROUPS || g->T > SK_GROUPED_MAX_ROWS) return SK_ERR_LIMIT;
  if (g->N > SK_GROUPED_MAX_ROWS || g->K > SK_GROUPED_MAX_ROWS) return SK_ERR_LIMIT;   // (room to round up to a tile)
  const bool tn = g->kind == SK_GROUPED_TN, nn = g->kind == SK_GROUPED_NN;
  const bool f32 = (g->flags & SK_FLAG_OUT_F32) != 0;
  if (f32 && !tn) return SK_ERR_ARG;
  if (g->lda < g->K || g->ldb < (g->kind == SK_GROUPED_NT ? g->K : g->N) || g->ldc < g->N) return SK_ERR_SHAPE;
  const long long b_rows = g->kind == SK_GROUPED_NT ? g->N : g->K;
  if (!tn && g->E > 1 && g->stride_b < b_rows * g->ldb) return SK_ERR_SHAPE;
  if (tn && g->E > 1 && g->stride_c < static_cast<long long>(g->K) * g->ldc) return SK_ERR_SHAPE;
  // TMA: 16-byte aligned bases and pitches
  if (!aligned(A, 16) || !aligned(B, 16) || (g->lda & 7) != 0 || (g->ldb & 7) != 0) return SK_ERR_ALIGN;
  if (!tn && g->E > 1 && (g->stride_b & 7) != 0) return SK_ERR_ALIGN;
  if (!aligned(C, f32 ? 4 : 2) || !aligned(offsets, (g->flags & SK_FLAG_OFFSETS_64) ? 8 : 4)) return SK_ERR_ALIGN;
  sk_problem any;
  memset(&any, 0, sizeof(any));
  any.num_sms = g->num_sms;
  int sms = 0, dev_sms = 0;
  int st = sk_resolve_grid(&any, &sms, &dev_sms);
  if (st != SK_OK) return st;
  if (sms < 2) return SK_ERR_LIMIT;   // CTA pairs
  if (!ws || ws_bytes < sk_ws_total_bytes(dev_sms)) return SK_ERR_WORKSPACE;
  if (!aligned(ws, 256)) return SK_ERR_ALIGN;

  GroupedParams p;
  memset(&p, 0, sizeof(p));
  p.T = g->T; p.E = g->E; p.N = g->N; p.K = g->K;
  p.ldc = g->ldc; p.stride_c = g->E > 1 ? g->stride_c : static_cast<long long>(g->K) * g->ldc;
  p.offsets = offsets;
  p.off64 = (g->flags & SK_FLAG_OFFSETS_64) ? 1 : 0;
  const bool bf16 = (g->flags & SK_FLAG_BF16) != 0;
  p.zero_rest = (g->flags & SK_FLAG_ZERO_REST) ? 1 : 0;
  p.timeout_ns = (g->timeout_us > 0 ? static_cast<unsigned long long>(g->timeout_us) : 2000000ULL) * 1000ULL;
  p.ws = sk_ws_carve(ws, dev_sms);
  st = sk_choose_status(g->flags, &p.ws);
  if (st != SK_OK) return st;
  const cudaStream_t cs = static_cast<cudaStream_t>(stream);
  const bool pdl = (g->flags & SK_FLAG_PDL) != 0;
  const uint64_t ldb = static_cast<uint64_t>(g->ldb), stride_b = g->E > 1 ? static_cast<uint64_t>(g->stride_b) : ldb * b_rows;
  static SkPerDeviceOnce attrs;
  cudaError_t e = attrs.run([]() {
    const void* kernels[15] = {
        reinterpret_cast<const void*>(sk_grouped_rows_kernel<false, false, false>),
        reinterpret_cast<const void*>(sk_grouped_rows_kernel<false, false, true>),
        reinterpret_cast<const void*>(sk_grouped_rows_kernel<false, true, false>),
        reinterpret_cast<const void*>(sk_grouped_rows_kernel<false, true, true>),
        reinterpret_cast<const void*>(sk_grouped_rows_kernel<true, false, false>),
        reinterpret_cast<const void*>(sk_grouped_rows_kernel<true, false, true>),
        reinterpret_cast<const void*>(sk_grouped_rows_kernel<true, true, false>),
        reinterpret_cast<const void*>(sk_grouped_rows_kernel<true, true, true>),
        reinterpret_cast<const void*>(sk_grouped_sum_kernel<OUT_F16, false, false>),
        reinterpret_cast<const void*>(sk_grouped_sum_kernel<OUT_F16, true, false>),
        reinterpret_cast<const void*>(sk_grouped_sum_kernel<OUT_BF16, false, false>),
        reinterpret_cast<const void*>(sk_grouped_sum_kernel<OUT_BF16, true, false>),
        reinterpret_cast<const void*>(sk_grouped_sum_kernel<OUT_F32, false, false>),
        reinterpret_cast<const void*>(sk_grouped_sum_kernel<OUT_F32, false, true>),
        reinterpret_cast<const void*>(sk_grouped_sum_kernel<OUT_F32, true, true>)};
    cudaError_t r = cudaSuccess;
    for (int i = 0; i < 15 && r == cudaSuccess; ++i)
      r = cudaFuncSetAttribute(kernels[i], cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_LIMIT);
    return r;
  });
  if (e != cudaSuccess) return sk_set_cuda_error(e);
  const int units = sms / 2;

  if (tn) {
    p.tiles_f = (g->K + 255) / 256;
    // Tiles of 256 columns of N, or of 128 while every one of those gets a pair of its own and the sums
    // are long (8 x 512 x 512 with 250 rows each: 11.2 us against 11.8 with 128)
    const bool longish = g->T / BK / g->E >= SUM_MIN_RUN;
    p.bn_max = longish && static_cast<long long>(p.tiles_f) * ((g->N + 127) / 128) * g->E <= units ? 128 : MAX_BN;
    p.tiles_n = (g->N + p.bn_max - 1) / p.bn_max;
    p.band = p.tiles_f < 8 ? p.tiles_f : 8;
    const long long total = static_cast<long long>(p.tiles_f) * p.tiles_n * g->E;
    if (total > (1LL << 30)) return SK_ERR_LIMIT;
    // Few tiles: up to four pairs per sum (the last to finish adds their parts; 2 x 256 x 256 with
    // 8000 rows each: 56.6 -> 27.7 us)
    // -- if a part of an average group's sum has steps enough
    p.parts = static_cast<int>(units / total < SK_MAX_PARTS ? units / total : SK_MAX_PARTS);
    if (p.parts < 2 || g->T / BK / g->E < 2 * SUM_MIN_RUN) p.parts = 1;
    p.d_band = sk_div_make(p.band * p.tiles_n);
    p.d_in = sk_div_make(p.band);
    p.d_last = sk_div_make(p.tiles_f % p.band ? p.tiles_f % p.band : p.band);
    const int esz = f32 ? 4 : 2;
    p.c_tma = aligned(C, 16) && (p.ldc * esz) % 16 == 0 && (p.stride_c * esz) % 16 == 0;
    p.c_flat = p.c_tma && p.ldc == g->N;
    // (24 groups of 42 rows, 4096 x 2048, bf16: 81 -> 70 us; 60 of 5, 1408 x 2048: 64 -> 58; over eight
    // results in turn)
    p.c_stream = sk_c_streams(static_cast<double>(g->E) * g->K * g->N * esz, g->T / BK / g->E);
    p.idesc = umma_idesc_f16(2 * HALF_M, 0, 1, bf16) | (1u << 15);   // both operands MN-major
    SumMaps maps;
    CUtensorMap tmC;
    memset(&tmC, 0, sizeof(tmC));
    for (int i = 0; i < 3 && st == SK_OK; ++i) {
      st = make_map(&maps.a[i], A, false, 0, g->T, g->K, g->lda, 0, 64, 16u << i);
      if (st == SK_OK) st = make_map(&maps.b[i], B, false, 0, g->T, g->N, ldb, 0, 64, 16u << i);
    }
    if (st == SK_OK && p.c_tma) st = make_map(&tmC, C, f32, g->E, g->K, g->N, p.ldc, p.stride_c, f32 ? 32 : 64, 32);
    if (st != SK_OK) return st;
    // Stages: as many as fit, six for up to 328 groups, five above.
    const int fixed = 1024 + EPI_WARPS * 4096 + CTRL_BYTES + table_bytes(g->E, false);
    p.stages = (SMEM_LIMIT - fixed) / TN_STEP;
    // fp32 results of short sums are bound by their stores, which do better with less read ahead of
    // them, or no worse: four, up to 2.5 steps per group (32 groups of 4096 x 2048: 100 rows 207 -> 202 us,
    // 64 and 128 rows the same within 1 %; 190 rows 211 -> 220; 32 uneven groups of 4099 rows in all, 2048 x 4096,
    // both gradients 340 -> 338)
    if (f32 && 2LL * g->T <= 5LL * BK * g->E && p.stages > 4) p.stages = 4;
    const int smem = fixed + p.stages * TN_STEP;
    const int grid = 2 * static_cast<int>(total * p.parts < units ? total * p.parts : units);
    const bool split = p.parts > 1;   // (fp32: then also long)
    const bool lengthy = g->T > SUM_RUN * BK;
    auto kernel = f32 ? (split ? sk_grouped_sum_kernel<OUT_F32, true, true>
                               : lengthy ? sk_grouped_sum_kernel<OUT_F32, false, true> : sk_grouped_sum_kernel<OUT_F32, false, false>)
                  : bf16 ? (split ? sk_grouped_sum_kernel<OUT_BF16, true, false> : sk_grouped_sum_kernel<OUT_BF16, false, false>)
                         : (split ? sk_grouped_sum_kernel<OUT_F16, true, false> : sk_grouped_sum_kernel<OUT_F16, false, false>);
    e = sk_launch(kernel, grid, TN_THREADS, smem, cs, 2, pdl, maps, tmC, C, p);
    return e == cudaSuccess ? SK_OK : sk_set_cuda_error(e);
  }

  const int t32 = g->T < MAX_BN ? (g->T + 31) & ~31 : MAX_BN;
  p.bn_max = t32;
  for (int j = 0; j < 4; ++j) p.d_rows[j] = sk_div_make(tile_rows(p.bn_max, j));
  p.tiles_f = (g->N + 255) / 256;
  // (row tiles: at most one ragged one per group besides the full ones)
  if ((static_cast<long long>(g->T) / p.bn_max + g->E + 1) * p.tiles_f > (1LL << 30)) return SK_ERR_LIMIT;
  p.c_vec_ok = aligned(C, 16) && (g->ldc & 7) == 0;
  p.c_words = aligned(C, 4) && (g->ldc & 1) == 0;
  // the box that a tile of bn_max rows loads, see the producer
  const int half = p.bn_max / 2;
  p.b_step_bytes = (half <= 16 ? 16 : half <= 64 ? 64 : 128) * 128;
  const int fixed = 1024 + CTRL_BYTES + EPI_WARPS * TURN_BYTES + table_bytes(g->E, true);
  // Stages of one step each, as many as fit (six for tiles of 256 rows, eleven for the fewest;
  // three of two steps were 2-5 % slower).
  p.stages = (SMEM_LIMIT - fixed) / (A_STEP_BYTES + p.b_step_bytes);
  if (p.stages > MAX_STAGES) p.stages = MAX_STAGES;
  const int smem = fixed + p.stages * (A_STEP_BYTES + p.b_step_bytes);
  p.idesc = umma_idesc_f16(2 * HALF_M, 0, 0, bf16) | (nn ? (1u << 15) : 0u);
  p.steps = (g->K + BK - 1) / BK;
  p.d_steps = sk_div_make(p.steps);
  // (measured: 4 rows, 512 features: 16 steps 8.2 us whole, 8.7 split; 32 steps 10.6 and 9.2)
  const bool split = p.steps >= 24 && 2 * p.tiles_f <= units;
  CUtensorMap tmW, tmX[3];
  st = nn ? make_map(&tmW, B, false, g->E, g->K, g->N, ldb, stride_b, 64, 64)
          : make_map(&tmW, B, false, g->E, g->N, g->K, ldb, stride_b, 64, HALF_M);
  const uint32_t boxes[3] = {16, 64, 128};
  memset(tmX, 0, sizeof(tmX));
  for (int i = 0; i < 3 && st == SK_OK; ++i)   // (only those that a tile can use)
    if (i == 0 || boxes[i - 1] < static_cast<uint32_t>(half))
      st = make_map(&tmX[i], A, false, 0, g->T, g->K, g->lda, 0, 64, boxes[i]);
  if (st != SK_OK) return st;
  const int grid = 2 * units;
  uint16_t* c = static_cast<uint16_t*>(C);
  auto kernel = nn ? (bf16 ? (split ? sk_grouped_rows_kernel<true, true, true> : sk_grouped_rows_kernel<true, true, false>)
                           : (split ? sk_grouped_rows_kernel<true, false, true> : sk_grouped_rows_kernel<true, false, false>))
                   : (bf16 ? (split ? sk_grouped_rows_kernel<false, true, true> : sk_grouped_rows_kernel<false, true, false>)
                           : (split ? sk_grouped_rows_kernel<false, false, true> : sk_grouped_rows_kernel<false, false, false>));
  e = sk_launch(kernel, grid, NT_THREADS, smem, cs, 2, pdl, tmW, tmX[0], tmX[1], tmX[2], c, p);
  return e == cudaSuccess ? SK_OK : sk_set_cuda_error(e);
}
