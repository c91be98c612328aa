// Products of many rows with 4-bit weights (format: int4.cuh) on the tcgen05 tensor cores, with the weights decoded on their
// way into tensor memory: the dense product Y = X W^T, and the two products of a mixture-of-experts layer over the rows
// of each expert.
//
// The problem is transposed, D^T[n, m] = sum_k W[n, k] X[m, k]: the instruction's M dimension is 256 weight rows of a CTA
// pair (cta_group::2), its N dimension up to 256 rows of X, A = W from tensor memory, B = X from shared memory.  A decoding
// thread owns one weight row = one tensor-memory lane; 64 columns of it are 32 registers and one tcgen05.st.
//
// Roles per CTA (512 threads, or 768 for tiles of up to 128 rows: see Shape):
//   warp 0       TMA producer of X: this CTA's half of the rows, boxes of 128 or 32 rows x 64 columns, SWIZZLE_128B
//   warp 1       pair leader: issues the MMAs and commits; other CTA: forwards "my operands are in place"
//   warp 2       producer of packed weights: whole tiles by TMA into a ring of its own
//   warps 4..7   epilogue
//   warps 8..    decoding; groups of four warps take the stages in turn
//
// Rows of a tile: 256 at most, rounded up to 32 for the instruction, so a short tile costs what it needs on the tensor pipe.
// Tensor memory: columns [0, 256) accumulator, [256 + 64 s, +64) A stage s (two 64-column steps).
// Schedule of the dense product: the K loops of all tiles are cut into units and dealt out evenly over the pairs.  Pieces of
// tiles go to the workspace in fp32 and a second kernel sums them in pair order: with 16 tiles over 74 pairs (256 x 4096 x
// 4096) a sum by the contributor that arrives last, 128 threads at two 32 KiB copies in flight, took 45 of 68 thousand
// cycles; a kernel of its own has all SMs for it.  Experts: whole tiles, dealt out in turn.
// What bounds it: with many rows the tensor pipe under the power limit (4096 x 14336 x 4096 fp16 345 us = 1.39 PFLOP/s with cool
// clocks, 413 us in a long run); with few rows the decoding warps' chain of waits and arithmetic (64 x 28672 x 8192 bf16 46 us =
// 2.6 TB/s of packed weights, where one more or less stage, four times fewer instructions on the tensor pipe or weights from L2 made
// no difference, and twice as many decoding warps took 57 to 46).
// Every wait is bounded; no TMA load uses cluster multicast.
#include "int4.cuh"
#include "tc_ptx.cuh"

namespace vqg {

using namespace tc;

namespace {

constexpr int kRows = 256;               // rows of X per tile, at most
constexpr int BNH = 128, BN = 256;       // weight rows per CTA and per pair
constexpr int BK = 64, KS = 2;           // columns per step, steps per stage
constexpr uint32_t kPStage = (BNH / 16) * KS * 512;       // 8 KiB of packed weights
constexpr uint32_t kTmemCols = 512, kStageCols = KS * BK / 2;

// What the kernel consists of for tiles of up to 256 rows of X, and of up to 128 (SHORT).  Decoding a stage is a chain of waits and
// of arithmetic that a warp does one after the other, some 900 cycles, whatever the rows; the epilogue of a short tile leaves the
// registers for twice as many warps that do it.
template <bool SHORT>
struct Shape {
  static constexpr int ROWS = SHORT ? 128 : kRows;
  static constexpr int STAGES = SHORT ? 6 : 4;
  static constexpr int GROUPS = SHORT ? 4 : 2;              // groups of four decoding warps, which take the stages in turn
  static constexpr int THREADS = 256 + 128 * GROUPS;
  static constexpr int OTHER_REGS = 40, EPILOGUE_REGS = SHORT ? 120 : 208;   // decoding: as launched, 80 or 128
  static constexpr uint32_t X_STEP = ROWS / 2 * BK * 2;     // half the rows x 64 columns
  static constexpr uint32_t X_STAGE = KS * X_STEP;
  static constexpr uint32_t PACKED = STAGES * X_STAGE;
  static constexpr uint32_t STAGING = PACKED + STAGES * kPStage;             // [256 rows][128 weight rows] of 16 bits, 128 of 32
  static constexpr uint32_t BARS = STAGING + kRows * BNH * 2;
  static constexpr uint32_t NUM_BARS = 4 * STAGES + 3;      // full, empty, packed full, packed empty; accumulator full, empty; epilogue
  static constexpr uint32_t TMEM_SLOT = BARS + (NUM_BARS + 1) / 2 * 16;
  static constexpr uint32_t SMEM = TMEM_SLOT + 16;
  static_assert(SMEM + 1024 <= 227 * 1024, "shared memory");
  static_assert(ROWS + STAGES * kStageCols <= kTmemCols, "tensor memory");
  static constexpr int LAUNCH_REGS = 65536 / THREADS / 8 * 8;
  static_assert(128 * (OTHER_REGS + EPILOGUE_REGS + GROUPS * LAUNCH_REGS) <= THREADS * LAUNCH_REGS, "registers of the launch");
};

enum { kDense = 0, kGated = 1, kDown = 2 };

struct TensorParams {
  Int4Weight w;
  void* y;
  int* status;
  int M;                     // dense: rows of X
  int m_tiles, n_tiles;
  int unit_stages, units_per_tile, q, r;   // see tensor3.cu
  float* ws_partial;         // [pair][piece][rank][256][128] fp32
  ExpertRows rows;
};

__device__ __forceinline__ int pair_begin(int b, int q, int r) { return b * q + (b < r ? b : r); }
__device__ __forceinline__ int pair_of_unit(int u, int q, int r) {
  const int big = r * (q + 1);
  return u < big ? u / (q + 1) : r + (u - big) / q;
}

struct Segment {
  int tile, kt_begin, kt_end, start;   // pipeline stages [kt_begin, kt_end) of the tile; first unit
  bool whole;
  int expert, row0, rows, n0;          // what the tile covers: rows of X, first weight row
};

// The pieces of a pair's share, in the order in which every role walks them.
template <int MODE>
struct Walk {
  int lo, hi, step;
  bool back_pending, front_first;
  __device__ __forceinline__ Walk(int pair, int n_pairs, const TensorParams& p) {
    if constexpr (MODE == kDense) {
      lo = pair_begin(pair, p.q, p.r);
      hi = pair_begin(pair + 1, p.q, p.r);
      back_pending = (hi % p.units_per_tile) != 0;
      front_first = (pair & 1) != 0 && (lo % p.units_per_tile) != 0;
    } else {
      lo = pair;
      hi = *p.rows.n_chunks * p.n_tiles;
      step = n_pairs;
    }
  }
  __device__ __forceinline__ bool next(Segment& g, const TensorParams& p) {
    if (lo >= hi) return false;
    const int stages = (p.w.k_tiles() + KS - 1) / KS;
    if constexpr (MODE == kDense) {
      bool rev = false;
      if (front_first) front_first = false;
      else if (back_pending) { rev = true; back_pending = false; }
      int end;
      if (!rev) {
        g.tile = lo / p.units_per_tile;
        g.start = lo;
        end = min(hi, (g.tile + 1) * p.units_per_tile);
        lo = end;
      } else {
        g.tile = (hi - 1) / p.units_per_tile;
        g.start = max(lo, g.tile * p.units_per_tile);
        end = hi;
        hi = g.start;
      }
      const int t0 = g.tile * p.units_per_tile;
      g.kt_begin = (g.start - t0) * p.unit_stages;
      g.kt_end = min((end - t0) * p.unit_stages, stages);
      g.whole = g.start == t0 && end == t0 + p.units_per_tile;
      g.expert = 0;
      g.row0 = (g.tile % p.m_tiles) * kRows;
      g.rows = min(kRows, p.M - g.row0);
      g.n0 = (g.tile / p.m_tiles) * BN;
    } else {
      g.tile = g.start = lo;
      lo += step;
      g.kt_begin = 0; g.kt_end = stages; g.whole = true;
      const int4 c = __ldg(p.rows.chunks + g.tile / p.n_tiles);
      g.expert = c.x; g.row0 = c.y; g.rows = c.z;
      g.n0 = (g.tile % p.n_tiles) * BN;
    }
    return true;
  }
};
// Weight row, within the CTA's 128, that tensor-memory lane 32 q + l holds.  Quarters 0 and 1 hold rows 0 ... 7 of the row tiles,
// whose codes are the low four bits of the bytes, quarters 2 and 3 rows 8 ... 15: the shifts of a decoding warp are then
// constants.  Eight neighbouring lanes are eight neighbouring rows.
__device__ __forceinline__ int row_of_lane(int q, int l) { return ((q & 1) * 4 + (l >> 3)) * 16 + (q >> 1) * 8 + (l & 7); }
__device__ __forceinline__ int mma_rows(int rows) { return (rows + 31) & ~31; }

__device__ __forceinline__ void mma_pair_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d), "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ bool elect_one() {
  uint32_t is;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(is));
  return is != 0;
}
// arrives at the barrier of both CTAs when the instructions so far are done
__device__ __forceinline__ void tc_commit_both(uint32_t bar) {
  asm volatile(
      "{\n\t.reg .b16 both;\n\tmov.b16 both, 3;\n\t"
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], both;\n\t}"
      ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tmem_st(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
        "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
        "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
      : "memory");
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack_pair(float a, float b) {
  if constexpr (BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

template <bool BF16, int MODE, bool SHORT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Shape<SHORT>::THREADS, 1)
int4_tensor_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_x32,
                   const __grid_constant__ CUtensorMap tmap_w, const TensorParams p) {
  using I = Int4Type<BF16>;
  using T = typename I::T;
  using C = Shape<SHORT>;
  constexpr int BM = C::ROWS, STAGES = C::STAGES;
  constexpr uint32_t kXStep = C::X_STEP, kXStage = C::X_STAGE, kPacked = C::PACKED, kStaging = C::STAGING, kBars = C::BARS, kAccCols = BM;
  extern __shared__ unsigned char smem_dyn[];
  const uint32_t raw = smem_u32(smem_dyn);
  const uint32_t base = (raw + 1023u) & ~1023u;
  unsigned char* base_ptr = smem_dyn + (base - raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int pair_id = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;
  const Int4Weight& w = p.w;

  auto bar_full = [&](int s) { return base + kBars + 8 * s; };
  auto bar_empty = [&](int s) { return base + kBars + 8 * (STAGES + s); };
  auto bar_pfull = [&](int s) { return base + kBars + 8 * (2 * STAGES + s); };
  auto bar_pempty = [&](int s) { return base + kBars + 8 * (3 * STAGES + s); };
  const uint32_t bar_acc_full = base + kBars + 8 * (4 * STAGES);
  const uint32_t bar_acc_empty = base + kBars + 8 * (4 * STAGES + 1);
  const uint32_t bar_epi = base + kBars + 8 * (4 * STAGES + 2);
  const uint32_t to_peer = map_to_cta(base, rank ^ 1u) - base;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(base_ptr + C::TMEM_SLOT);

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      // full: X has landed (one arrival and its bytes), four decoding warps have written their columns; in the leader one
      // more arrival says the same of the other CTA
      mbar_init(bar_full(s), 1 + 4 + (rank == 0 ? 1 : 0));
      mbar_init(bar_empty(s), 1);
      mbar_init(bar_pfull(s), 1);
      mbar_init(bar_pempty(s), 4);
    }
    mbar_init(bar_acc_full, 1);
    mbar_init(bar_acc_empty, 8);
    mbar_init(bar_epi, 4);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_smem();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(base + C::TMEM_SLOT), "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  grid_release();
  grid_wait();

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::OTHER_REGS));
    if (warp == 0) {
      // ------------------------------- X producer ---------------------------------------------
      // the whole warp walks; lane u * boxes + b issues one box (a single lane would need longer than a stage takes)
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      Walk<MODE> walk(pair_id, n_pairs, p);
      Segment g;
      while (ok && walk.next(g, p)) {
        const int half = mma_rows(g.rows) / 2;
        const int boxes = BM > 128 && half > 64 ? 1 : (half + 31) / 32;       // one box of 128 rows, or one or two of 32
        const CUtensorMap* map = BM > 128 && half > 64 ? &tmap_x : &tmap_x32;
        const int box_rows = BM > 128 && half > 64 ? 128 : 32;
        const int u = lane / boxes, b = lane % boxes;
        const int row = g.row0 + static_cast<int>(rank) * half + 32 * b;
        for (int kt = g.kt_begin; kt < g.kt_end; ++kt) {
          if (!(ok = mbar_wait_cluster(bar_empty(stage), phase ^ 1, p.status, DS_STAGE_EMPTY_TIMEOUT))) break;
          if (lane == 0) mbar_expect_tx(bar_full(stage), KS * boxes * box_rows * (BK * 2));
          __syncwarp();
          if (u < KS) tma_load_2d(base + stage * kXStage + u * kXStep + b * 4096, map, (kt * KS + u) * BK, row, bar_full(stage));
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
      }
    } else if (warp == 1) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      Walk<MODE> walk(pair_id, n_pairs, p);
      Segment g;
      if (rank == 0) {
        // ------------------------------- MMA issuer -------------------------------------------
        // The whole warp walks and one lane issues: what the instructions take is then the same in all lanes, and the compiler
        // keeps it where they want it.
        const uint32_t d_t = __shfl_sync(0xffffffffu, tmem_base, 0);
        uint32_t acc_phase = 0;
        while (ok && walk.next(g, p)) {
          // A and B of type fp16 (0) or bf16 (1), D fp32, both K-major
          const uint32_t idesc = (1u << 4) | (BF16 ? (1u << 7) | (1u << 10) : 0u) |
                                 (static_cast<uint32_t>(mma_rows(g.rows) >> 3) << 17) | (static_cast<uint32_t>(BN >> 4) << 24);
          ok = __all_sync(0xffffffffu, mbar_wait_cluster(bar_acc_empty, acc_phase ^ 1, p.status, DS_ACC_EMPTY_TIMEOUT));
          if (!ok) break;
          tc_fence_after();
          for (int kt = g.kt_begin; kt < g.kt_end; ++kt) {
            ok = __all_sync(0xffffffffu, mbar_wait_cluster(bar_full(stage), phase, p.status, DS_TMA_FULL_TIMEOUT));
            if (!ok) break;
            tc_fence_after();
            if (elect_one()) {
              const uint32_t a_t = d_t + kAccCols + static_cast<uint32_t>(stage) * kStageCols;
#pragma unroll
              for (int u = 0; u < KS; ++u) {
                const uint64_t bd = make_desc(base + stage * kXStage + u * kXStep);
#pragma unroll
                for (int k = 0; k < BK / 16; ++k)
                  mma_pair_ts(d_t, a_t + u * (BK / 2) + 8 * k, bd + 2 * k, idesc, ((kt - g.kt_begin) | u | k) != 0 ? 1u : 0u);
              }
              tc_commit_both(bar_empty(stage));
              if (kt + 1 == g.kt_end) tc_commit_both(bar_acc_full);
            }
            __syncwarp();
            if (++stage == STAGES) { stage = 0; phase ^= 1; }
          }
          acc_phase ^= 1;
        }
      } else if (lane == 0) {
        // ------------------------------- forwarder --------------------------------------------
        while (ok && walk.next(g, p)) {
          for (int kt = g.kt_begin; kt < g.kt_end; ++kt) {
            if (!(ok = mbar_wait(bar_full(stage), phase, p.status, DS_TMA_FULL_TIMEOUT))) break;
            mbar_arrive_remote(bar_full(stage) + to_peer);
            if (++stage == STAGES) { stage = 0; phase ^= 1; }
          }
        }
      }
    } else if (warp == 2) {
      // ------------------------------- packed-weight producer -----------------------------------
      // one copy per stage: eight row tiles x KS column tiles.  Row tiles behind the last one are another expert's, or zero.
      if (lane == 0) {
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        Walk<MODE> walk(pair_id, n_pairs, p);
        Segment g;
        while (ok && walk.next(g, p)) {
          const int tile0 = g.expert * w.row_tiles() + (g.n0 + static_cast<int>(rank) * BNH) / 16;
          for (int kt = g.kt_begin; kt < g.kt_end; ++kt) {
            if (!(ok = mbar_wait(bar_pempty(stage), phase ^ 1, p.status, DS_STAGE_EMPTY_TIMEOUT))) break;
            mbar_expect_tx(bar_pfull(stage), kPStage);
            tma_load_3d(base + kPacked + stage * kPStage, &tmap_w, 0, kt * KS, tile0, bar_pfull(stage));
            if (++stage == STAGES) { stage = 0; phase ^= 1; }
          }
        }
      }
    }
  } else if (warp < 8) {
    // ------------------------------- epilogue -----------------------------------------------------
    // lane = weight row, column = row of X
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::EPILOGUE_REGS));
    const int quarter = warp & 3, my_row = row_of_lane(quarter, lane);
    uint32_t acc_phase = 0, epi_phase = 0;
    bool ok = true;
    const uint32_t leader_acc_empty = bar_acc_empty + (rank == 0 ? 0u : to_peer);
    unsigned char* stg = base_ptr + kStaging;
    auto epi_sync = [&]() -> bool {
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_epi);
      const bool done = mbar_wait(bar_epi, epi_phase, p.status, DS_EPILOGUE_SYNC_TIMEOUT);
      epi_phase ^= 1;
      return done;
    };
    auto release = [&]() {   // tensor memory has been read: the next tile may overwrite it
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_remote(leader_acc_empty);
    };
    constexpr int OUT_COLS = MODE == kGated ? BNH / 2 : BNH;   // output columns of this CTA's half tile
    constexpr int ROW_BYTES = OUT_COLS * 2;
    constexpr size_t kPartialFloats = static_cast<size_t>(kRows) * BNH;
    Walk<MODE> walk(pair_id, n_pairs, p);
    Segment g;
    while (ok && walk.next(g, p)) {
      const int n0 = g.n0 + static_cast<int>(rank) * BNH;      // first weight row of this CTA
      const int cols = mma_rows(g.rows);
      if (!(ok = mbar_wait_cluster(bar_acc_full, acc_phase, p.status, DS_ACC_FULL_TIMEOUT))) break;
      tc_fence_after();
      acc_phase ^= 1;
      const uint32_t t_row = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
      if constexpr (MODE == kDown) {
        // fp32 rows of the slots.  Rows 128 ... 255 of X wait in registers while rows 0 ... 127 go to the staging tile, so that
        // tensor memory is free after one reading of it; each row leaves shared memory as one bulk copy of up to 512 bytes, which
        // the stores of the next tile's accumulation do not wait for.  (Stores from the registers, a row address each, kept the
        // accumulator for 12 to 19 thousand cycles per tile.)
        float* part = static_cast<float*>(p.y) + n0;
        const uint32_t bytes = n0 < w.N ? min(BNH, w.N - n0) * 4 : 0;     // a multiple of 128
        float* col = reinterpret_cast<float*>(stg) + my_row;
        auto send = [&](int first) {       // rows first ... first + 127 of the tile, one per lane
          fence_async_smem();
          if (!(ok = epi_sync())) return;
          const int m = first + quarter * 32 + lane;
          if (m < g.rows && bytes) {
            const int slot = __ldg(p.rows.row_slot + g.row0 + m);
            asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;"
                         ::"l"(part + static_cast<long long>(slot) * w.N), "r"(base + kStaging + (quarter * 32 + lane) * 512), "r"(bytes) : "memory");
          }
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        };
        auto sent = [&]() {                // the staging tile has been read
          asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
          ok = epi_sync();
        };
        uint32_t late[4][32];
        if (BM > 128 && cols > 128) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (128 + 32 * i < cols) tmem_ld32_async(t_row + 128 + 32 * i, late[i]);
        }
#pragma unroll 1
        for (int c = 0; c < min(cols, 128); c += 32) {
          uint32_t r[32];
          tmem_ld32_async(t_row + c, r);
          tmem_ld_wait(r);
#pragma unroll
          for (int j = 0; j < 32; ++j) col[(c + j) * BNH] = __uint_as_float(r[j]);
        }
        if constexpr (BM > 128) {
#pragma unroll
          for (int i = 0; i < 4; ++i) tmem_ld_wait(late[i]);
        }
        release();
        send(0);
        if (BM > 128 && ok && cols > 128) {
          sent();
          if (ok) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (128 + 32 * i < cols) {
#pragma unroll
                for (int j = 0; j < 32; ++j) col[(32 * i + j) * BNH] = __uint_as_float(late[i][j]);
              }
            send(128);
          }
        }
        if (ok) sent();
        if (!ok) break;
        continue;
      } else {
        if (g.whole) {
          if constexpr (MODE == kGated) {
            // Lanes 2i and 2i + 1 hold gate and up of output column i.  One exchange per two rows of X: the even lane finishes the
            // first, the odd lane the second.  The results wait in registers, two to one, until tensor memory is handed back.
            uint32_t hp[BM / 4];
            uint32_t qa[16], qb[16];
            const bool odd = (lane & 1) != 0;
            auto finish = [&](const uint32_t (&q)[16], uint32_t* out) {
#pragma unroll
              for (int j = 0; j < 16; j += 4) {
                float v[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                  const float first = __uint_as_float(q[j + 2 * i]), second = __uint_as_float(q[j + 2 * i + 1]);
                  const float recv = __shfl_xor_sync(0xffffffffu, odd ? first : second, 1);
                  v[i] = silu_mul(odd ? recv : first, odd ? second : recv);
                }
                out[j / 4] = pack_pair<BF16>(v[0], v[1]);
              }
            };
            tmem_ld16_async(t_row, qa);
#pragma unroll
            for (int c = 0; c < BM / 16; c += 2) {
              if (c * 16 < cols) {
                tmem_ld_wait16(qa);
                tmem_ld16_async(t_row + (c + 1) * 16, qb);
                finish(qa, hp + c * 4);
                tmem_ld_wait16(qb);
                if (c * 16 + 32 < cols) tmem_ld16_async(t_row + (c + 2) * 16, qa);
                else release();
                finish(qb, hp + (c + 1) * 4);
              }
            }
            unsigned short* col = reinterpret_cast<unsigned short*>(stg) + (my_row >> 1) + (odd ? OUT_COLS : 0);
#pragma unroll
            for (int q = 0; q < BM / 4; ++q) {
              if (4 * q < cols) {
                col[(4 * q) * OUT_COLS] = static_cast<unsigned short>(hp[q] & 0xffffu);
                col[(4 * q + 2) * OUT_COLS] = static_cast<unsigned short>(hp[q] >> 16);
              }
            }
          } else {
            // the whole row is converted in registers and tensor memory handed back before the first store
            uint32_t hp[BM / 2];
            uint32_t qa[16], qb[16];
            tmem_ld16_async(t_row, qa);
#pragma unroll
            for (int c = 0; c < BM / 16; c += 2) {
              if (c * 16 < cols) {
                tmem_ld_wait16(qa);
                tmem_ld16_async(t_row + (c + 1) * 16, qb);
#pragma unroll
                for (int j = 0; j < 8; ++j) hp[c * 8 + j] = pack_pair<BF16>(__uint_as_float(qa[2 * j]), __uint_as_float(qa[2 * j + 1]));
                tmem_ld_wait16(qb);
                if (c * 16 + 32 < cols) tmem_ld16_async(t_row + (c + 2) * 16, qa);
                else release();
#pragma unroll
                for (int j = 0; j < 8; ++j) hp[(c + 1) * 8 + j] = pack_pair<BF16>(__uint_as_float(qb[2 * j]), __uint_as_float(qb[2 * j + 1]));
              }
            }
            unsigned short* col = reinterpret_cast<unsigned short*>(stg) + my_row;
#pragma unroll
            for (int q = 0; q < BM / 2; ++q) {
              if (2 * q < cols) {
                col[(2 * q) * 128] = static_cast<unsigned short>(hp[q] & 0xffffu);
                col[(2 * q + 1) * 128] = static_cast<unsigned short>(hp[q] >> 16);
              }
            }
          }
        } else {
          const int slot = (g.start > g.tile * p.units_per_tile) ? 0 : 1;
          float* part = p.ws_partial + ((static_cast<size_t>(pair_id) * 2 + slot) * 2 + rank) * kPartialFloats + quarter * 32 + lane;
#pragma unroll 1
          for (int c = 0; c < cols; c += 32) {
            uint32_t r[32];
            tmem_ld32(t_row + c, r);
            if (c + 32 >= cols) release();
#pragma unroll
            for (int j = 0; j < 32; ++j) __stcg(part + static_cast<size_t>(c + j) * BNH, __uint_as_float(r[j]));
          }
          continue;                        // int4_tensor_sum_kernel adds the pieces up
        }
        if (!(ok = epi_sync())) break;   // the whole tile is in shared memory
        const int out_n = MODE == kGated ? w.N / 2 : w.N, out0 = MODE == kGated ? n0 / 2 : n0;
        T* out = static_cast<T*>(p.y);
        if (out_n % 8 == 0) {
          constexpr int LPR = ROW_BYTES / 16, RPW = 32 / LPR;
          const int rsel = lane / LPR, chunk = lane % LPR, ncol = out0 + chunk * 8;
#pragma unroll 4
          for (int m = quarter * RPW + rsel; m < g.rows; m += 4 * RPW)
            if (ncol < out_n)
              *reinterpret_cast<uint4*>(out + static_cast<long long>(g.row0 + m) * out_n + ncol) =
                  *reinterpret_cast<const uint4*>(stg + m * ROW_BYTES + chunk * 16);
        } else {   // rows that do not begin on 16 bytes: two bytes per lane, 32 neighbours together
          for (int m = quarter; m < g.rows; m += 4)
            for (int c = lane; c < OUT_COLS && out0 + c < out_n; c += 32)
              out[static_cast<long long>(g.row0 + m) * out_n + out0 + c] = reinterpret_cast<const T*>(stg + m * ROW_BYTES)[c];
        }
        if (!(ok = epi_sync())) break;   // the staging tile is rewritten by the next one
      }
    }
    if constexpr (MODE == kDown) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");   // every copy is complete
  } else {
    // ------------------------------- decoding -----------------------------------------------------
    // A warp takes every second or fourth stage whole: the waits, the handing over and the scales' bookkeeping of a stage take as long as the
    // arithmetic of one of its steps.
    constexpr int GROUPS = C::GROUPS;
    const int quarter = warp & 3, group = (warp - 8) >> 2;
    const int r = row_of_lane(quarter, lane);                  // weight row in the CTA
    const uint32_t src = base + kPacked + (r / 16) * (KS * 512) + (r & 7) * 16;
    const uint32_t a_lane = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + kAccCols;
    uint32_t done = 0;                                         // stages before the segment
    bool ok = true;
    Walk<MODE> walk(pair_id, n_pairs, p);
    Segment g;
    const bool halves = w.group == 32;                         // columns 0 ... 31 and 32 ... 63 of a step have scales of their own
    const bool whole = w.group % (KS * BK) == 0;               // the steps of a stage share theirs
    while (ok && walk.next(g, p)) {
      const int n = g.n0 + static_cast<int>(rank) * BNH + r;
      const uint32_t twice = n < w.N ? 0x10001u : 0u;
      // Scales and zero points, two of the warp's stages ahead and as loaded: nothing is computed from them before the stage in hand
      // is done, or the warp would wait for memory here.  Rows and columns that do not exist read the last ones and get a scale of
      // zero, so that no fill reaches a sum.
      const int nc = min(n, w.N - 1);
      const unsigned short* sc = static_cast<const unsigned short*>(w.scales) + g.expert * w.expert_scales() + nc;
      const uint8_t* ze = w.zeros ? w.zeros + g.expert * w.expert_scales() + nc : nullptr;
      struct Raw {
        unsigned short s[KS][2];
        uint8_t z[KS][2];
      };
      auto fetch = [&](Raw& f, int kt) {   // only the loads: a copy of what is on its way would wait for it
#pragma unroll
        for (int u = 0; u < KS; ++u)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if ((u == 0 || !whole) && (h == 0 || halves)) {
              const int at = int4_group_of(w, min((kt * KS + u) * BK + 32 * h, w.K - 32)) * w.N;
              f.s[u][h] = __ldg(sc + at);
              if (ze) f.z[u][h] = __ldg(ze + at);
            }
      };
      const uint32_t first = done - static_cast<uint32_t>(g.kt_begin);      // stage of column tile kt: first + kt
      int kt = g.kt_begin + static_cast<int>((static_cast<uint32_t>(group) - done) % GROUPS);
      done += static_cast<uint32_t>(g.kt_end - g.kt_begin);
      // one stage; f holds its scales and gets those of the stage after the warp's next one
      auto decode = [&](Raw& f, int kt) -> bool {
        const uint32_t it = first + static_cast<uint32_t>(kt), stage = it % STAGES, phase = (it / STAGES) & 1u;
        uint32_t s2[KS][2], off[KS][2];
        auto offset = [&](int zero) { return quarter < 2 ? I::offset(zero) : int4_offset_hi<BF16>(zero); };
        if (whole && (kt + 1) * (KS * BK) <= w.K) {            // (a few instructions instead of some eighty in a row)
          const uint32_t scale = f.s[0][0] * twice, o = ze ? offset(f.z[0][0] & 15) : offset(8);
#pragma unroll
          for (int i = 0; i < 2 * KS; ++i) { s2[i >> 1][i & 1] = scale; off[i >> 1][i & 1] = o; }
        } else {
#pragma unroll
          for (int u = 0; u < KS; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t scale = whole ? f.s[0][0] : halves ? f.s[u][h] : f.s[u][0];
              const int zero = !ze ? 8 : (whole ? f.z[0][0] : halves ? f.z[u][h] : f.z[u][0]) & 15;
              s2[u][h] = (kt * KS + u) * BK + 32 * h < w.K ? scale * twice : 0u;
              off[u][h] = offset(zero);
            }
        }
        fetch(f, kt + 2 * GROUPS);
        if (!mbar_wait(bar_pfull(stage), phase, p.status, DS_TMA_FULL_TIMEOUT)) return false;
        // pieces of a step: a whole one, with all codes read ahead, or half of one where there are fewer registers
        constexpr int WORDS = SHORT ? 8 : 16, PIECES = KS * 16 / WORDS;
        uint32_t codes[SHORT ? 1 : PIECES][WORDS];
        auto read = [&](uint32_t (&c)[WORDS], int piece) {
#pragma unroll
          for (int t = 0; t < WORDS / 4; ++t)
            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                         : "=r"(c[4 * t]), "=r"(c[4 * t + 1]), "=r"(c[4 * t + 2]), "=r"(c[4 * t + 3])
                         : "r"(src + stage * kPStage + piece * WORDS / 16 * 512 + (piece * WORDS % 16 / 4 + t) * 128));
        };
        if constexpr (!SHORT)
#pragma unroll
          for (int i = 0; i < PIECES; ++i) read(codes[i], i);
#pragma unroll
        for (int piece = 0; piece < PIECES; ++piece) {
          const int u = piece * WORDS / 16, w0 = piece * WORDS % 16;
          uint32_t (&c)[WORDS] = codes[SHORT ? 0 : piece];
          if constexpr (SHORT) read(c, piece);
          uint32_t a[2 * WORDS];
          if (quarter < 2) {
#pragma unroll
            for (int i = 0; i < WORDS; ++i) {
              a[2 * i] = int4_pair<BF16, 0, 0>(c[i], off[u][(w0 + i) >> 3], s2[u][(w0 + i) >> 3]);
              a[2 * i + 1] = int4_pair<BF16, 0, 1>(c[i], off[u][(w0 + i) >> 3], s2[u][(w0 + i) >> 3]);
            }
          } else {
#pragma unroll
            for (int i = 0; i < WORDS; ++i) {
              a[2 * i] = int4_pair_hi<BF16, 0>(c[i], off[u][(w0 + i) >> 3], s2[u][(w0 + i) >> 3]);
              a[2 * i + 1] = int4_pair_hi<BF16, 1>(c[i], off[u][(w0 + i) >> 3], s2[u][(w0 + i) >> 3]);
            }
          }
          if (piece == 0) {
            if (!mbar_wait_cluster(bar_empty(stage), phase ^ 1, p.status, DS_STAGE_EMPTY_TIMEOUT)) return false;
            tc_fence_after();
          }
          __syncwarp();
          tmem_st(a_lane + stage * kStageCols + piece * WORDS * 2, a);
        }
        if (lane == 0) mbar_arrive(bar_pempty(stage));
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_full(stage));
        return true;
      };
      // (two sets of scales in turn, not one handed to the other: a move would wait for the load)
      Raw even{}, odd{};
      fetch(even, kt);
      fetch(odd, kt + GROUPS);
      while (kt < g.kt_end) {
        if (!(ok = decode(even, kt))) break;
        kt += GROUPS;
        if (kt >= g.kt_end) break;
        if (!(ok = decode(odd, kt))) break;
        kt += GROUPS;
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols) : "memory");
  }
}

// Sums the pieces of the tiles that several pairs shared, in pair order.  blockIdx.y = pair: the tile that its range ends inside,
// if this pair is the first to work on it; blockIdx.x and the thread: rank, row of X, four neighbouring weight rows.
template <bool BF16>
__global__ void __launch_bounds__(256)
int4_tensor_sum_kernel(const TensorParams p) {
  using I = Int4Type<BF16>;
  using T = typename I::T;
  grid_release();
  grid_wait();
  const int end = pair_begin(blockIdx.y + 1, p.q, p.r);
  if (end % p.units_per_tile == 0) return;
  const int tile = end / p.units_per_tile, t0u = tile * p.units_per_tile;
  const int b_first = pair_of_unit(t0u, p.q, p.r), b_last = pair_of_unit(t0u + p.units_per_tile - 1, p.q, p.r);
  if (b_first != static_cast<int>(blockIdx.y)) return;
  const int i = blockIdx.x * 256 + threadIdx.x;
  const int lane4 = (i & 31) * 4, rank = (i >> 5) & 1, m = i >> 6;
  const int row0 = (tile % p.m_tiles) * kRows, n = (tile / p.m_tiles) * BN + rank * BNH + row_of_lane(lane4 >> 5, lane4 & 31);
  if (m >= kRows || row0 + m >= p.M || n >= p.w.N) return;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int b = b_first; b <= b_last; ++b) {
    const int piece = pair_begin(b, p.q, p.r) > t0u ? 0 : 1;
    const float4 v = __ldcg(reinterpret_cast<const float4*>(
        p.ws_partial + ((static_cast<size_t>(b) * 2 + piece) * 2 + rank) * (static_cast<size_t>(kRows) * BNH) + static_cast<size_t>(m) * BNH + lane4));
    sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
  }
  T* out = static_cast<T*>(p.y) + static_cast<long long>(row0 + m) * p.w.N + n;
  if (p.w.N % 4 == 0) {
    *reinterpret_cast<uint2*>(out) = make_uint2(pack_pair<BF16>(sum.x, sum.y), pack_pair<BF16>(sum.z, sum.w));
  } else {
    const float v[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (n + c < p.w.N) out[c] = I::from_float(v[c]);
  }
}

// Rows of X in the order of the plan (one block per row).
__global__ void __launch_bounds__(128)
gather_rows_kernel(const uint4* __restrict__ x, const ExpertRows rows, uint4* __restrict__ out, int vecs) {
  grid_release();
  grid_wait();
  for (int r = blockIdx.x; r < rows.n_chunks[1]; r += gridDim.x) {
    const uint4* src = x + static_cast<long long>(rows.row_slot[r] / rows.top_k) * vecs;
    for (int i = threadIdx.x; i < vecs; i += blockDim.x) out[static_cast<long long>(r) * vecs + i] = __ldg(src + i);
  }
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encode_fn() {
  static EncodeFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<EncodeFn>(f);
  }();
  return fn;
}
// 16-bit row-major [rows, cols], box of box_rows rows x 64 columns, zero fill (the columns that fill up the last step among it)
bool make_x_map(CUtensorMap* map, const void* ptr, int rows, int cols, int box_rows, bool bf16) {
  EncodeFn fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(cols) * 2};
  const cuuint32_t box[2] = {BK, static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t estr[2] = {1, 1};
  return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(ptr), dims,
            strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// packed weights as [row tiles][column tiles][128 words], box of a stage of a CTA: whole tiles
bool make_w_map(CUtensorMap* map, const Int4Weight& w, int experts) {
  EncodeFn fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t k = w.k_tiles();
  const cuuint64_t dims[3] = {128, k, static_cast<cuuint64_t>(w.row_tiles()) * experts}, strides[2] = {512, k * 512};
  const cuuint32_t box[3] = {128, KS, BNH / 16}, estr[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, const_cast<uint8_t*>(w.packed), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
int sm_pairs() { return max(1, sm_count_cached() / 2); }
constexpr size_t kPairPartialBytes = 2 * 2 * static_cast<size_t>(kRows) * BNH * sizeof(float);

template <bool BF16, int MODE, bool SHORT>
int launch_shape(int pairs, const void* x, int rows, const TensorParams& p, cudaStream_t s) {
  static SmemOptIn opt_in;
  auto kernel = int4_tensor_kernel<BF16, MODE, SHORT>;
  CUtensorMap map, map32, map_w;
  if (!make_x_map(&map, x, rows, p.w.K, 128, BF16) || !make_x_map(&map32, x, rows, p.w.K, 32, BF16) ||
      !make_w_map(&map_w, p.w, MODE == kDense ? 1 : p.rows.E) || !opt_in.ask(kernel))
    return VQG_ERR_LAUNCH;
  return cuda_status(launch_ahead(kernel, dim3(2 * pairs), Shape<SHORT>::THREADS, Shape<SHORT>::SMEM + 1024, s, false, map, map32, map_w, p));
}

template <int MODE>
int launch(int pairs, const void* x, int rows, bool is_short, bool bf16, const TensorParams& p, cudaStream_t s) {
  if (is_short) return bf16 ? launch_shape<true, MODE, true>(pairs, x, rows, p, s) : launch_shape<false, MODE, true>(pairs, x, rows, p, s);
  return bf16 ? launch_shape<true, MODE, false>(pairs, x, rows, p, s) : launch_shape<false, MODE, false>(pairs, x, rows, p, s);
}

}  // namespace

size_t int4_tensor_workspace_bytes() {
  return static_cast<size_t>(sm_pairs()) * kPairPartialBytes;
}

int launch_int4_tensor(const Int4Weight& w, const void* x, void* y, int M, bool bf16, void* ws, size_t ws_bytes, cudaStream_t s) {
  TensorParams p{};
  p.w = w; p.y = y; p.M = M;
  p.status = device_status_ptr();
  p.m_tiles = (M + kRows - 1) / kRows;
  p.n_tiles = (w.N + BN - 1) / BN;
  const int max_pairs = sm_pairs(), stages = (w.k_tiles() + KS - 1) / KS;
  const long long tiles = static_cast<long long>(p.m_tiles) * p.n_tiles;
  if (tiles > 0x7fffffffLL / (stages + 1)) return VQG_ERR_UNSUPPORTED;
  const bool split = ws && reinterpret_cast<uintptr_t>(ws) % 256 == 0 &&
                     ws_bytes >= static_cast<size_t>(max_pairs) * kPairPartialBytes && stages > 1 &&
                     tiles % max_pairs != 0;
  p.unit_stages = split ? (stages >= 8 ? 2 : 1) : stages;
  p.units_per_tile = (stages + p.unit_stages - 1) / p.unit_stages;
  const long long units = tiles * p.units_per_tile;
  const int pairs = units < max_pairs ? static_cast<int>(units) : max_pairs;
  p.q = static_cast<int>(units / pairs);
  p.r = static_cast<int>(units % pairs);
  p.ws_partial = split ? static_cast<float*>(ws) : nullptr;
  const int st = launch<kDense>(pairs, x, M, M <= Shape<true>::ROWS, bf16, p, s);
  if (st != VQG_OK || !split || pairs == 1) return st;
  const dim3 grid(((M < kRows ? M : kRows) * 64 + 255) / 256, pairs - 1);
  return cuda_status(bf16 ? launch_ahead(int4_tensor_sum_kernel<true>, grid, 256, 0, s, false, p)
                          : launch_ahead(int4_tensor_sum_kernel<false>, grid, 256, 0, s, false, p));
}

namespace {
int launch_experts(const Int4Weight& w, const void* x, void* y, const ExpertRows& rows, int chunk_rows, int max_chunks, bool bf16, bool gated,
                   cudaStream_t s) {
  TensorParams p{};
  p.w = w; p.y = y; p.rows = rows;
  p.status = device_status_ptr();
  p.n_tiles = (w.N + BN - 1) / BN;
  const long long most = static_cast<long long>(max_chunks) * p.n_tiles;
  if (most > 0x7fffffffLL) return VQG_ERR_UNSUPPORTED;
  const int pairs = most < sm_pairs() ? static_cast<int>(most) : sm_pairs();
  const bool is_short = chunk_rows <= Shape<true>::ROWS;
  return gated ? launch<kGated>(pairs, x, rows.slots, is_short, bf16, p, s) : launch<kDown>(pairs, x, rows.slots, is_short, bf16, p, s);
}
}  // namespace

int launch_int4_tensor_gated(const Int4Weight& w, const void* x_rows, void* h, const ExpertRows& rows, int chunk_rows, int max_chunks, bool bf16,
                             cudaStream_t s) {
  return launch_experts(w, x_rows, h, rows, chunk_rows, max_chunks, bf16, true, s);
}
int launch_int4_tensor_down(const Int4Weight& w, const void* h, float* part, const ExpertRows& rows, int chunk_rows, int max_chunks, bool bf16,
                            cudaStream_t s) {
  return launch_experts(w, h, part, rows, chunk_rows, max_chunks, bf16, false, s);
}

int launch_gather_rows(const void* x, const ExpertRows& rows, void* out, int cols, cudaStream_t s) {
  const int blocks = rows.slots < 148 * 16 ? rows.slots : 148 * 16;
  return cuda_status(launch_ahead(gather_rows_kernel, dim3(blocks), 128, 0, s, false, static_cast<const uint4*>(x), rows,
                                  static_cast<uint4*>(out), cols / 8));
}

}  // namespace vqg
