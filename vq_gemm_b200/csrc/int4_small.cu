// Products of a few rows with 4-bit weights (format: int4.cuh): Y[m, n] = sum_k X[m, k] W[n, k], and the two products of
// the experts of a mixture-of-experts layer over the rows that chose them.
//
// A warp takes blocks of B neighbouring 64-column steps of R row tiles (16 weight rows each).  A lane's 16 bytes of a tile give the
// A fragments of four mma.sync m16n8k16, whose B fragments are 32 consecutive bytes of a row of X.  Every warp copies its tiles
// asynchronously into a ring of its own in shared memory, SLOTS blocks ahead: no warp waits for another, and no register or
// scoreboard is tied up by a load from memory.  The copies go in memory order, lane i the i-th 16 bytes (in the order in
// which the lanes need them a quarter warp would touch four lines instead of one, which alone cost 14 of 46 us at 1 x
// 28672 x 8192), into places that are swizzled so that neither side has bank conflicts: see place().  The sums of a team
// of warps (two, four or eight, see below) meet in shared memory.
//
// What bounds it: bytes by the count (half a byte per weight and nothing twice), issue and latency by measurement.  1 x 28672 x
// 8192 bf16 takes 36.9 us, 3.3 TB/s where a copy reaches 6.5: some 106 instructions of a warp per tile of 16 x 64 weights, half of
// them the decoding (mask, subtract, multiply: each weight is rounded to T as the format says), 64 % of the issue slots busy.
// 1 x 4096 x 4096 takes 5.2 us, 16 x 11008 x 4096 14.0.
#include <type_traits>

#include "int4.cuh"

namespace vqg {
namespace {

constexpr int kWarps = 16;                   // of a block of the direct down product
constexpr size_t kSmallSmem = 227 * 1024;    // shared memory of a block, at most

struct SmallParams {
  Int4Weight w;
  const void* x;
  void* y;
  int M, chunks;             // chunks: of the dense product; for experts at most as many
  ExpertRows rows;
};

enum { kDense = 0, kGated = 1, kDown = 2 };

template <bool BF16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Scales and zero points of rows g and g + 8 of R row tiles for B steps, one for every SPAN steps (2 where a group is a multiple
// of 128 columns), as loaded.
template <bool ZEROS, int R, int B, int SPAN>
struct Scales {
  static constexpr int S = B / SPAN;
  unsigned short s_lo[S][R], s_hi[S][R];
  uint8_t z_lo[ZEROS ? S : 1][R], z_hi[ZEROS ? S : 1][R];
};

// One expert's weight as a lane sees it.
struct View {
  const uint8_t* packed;
  const unsigned short* scales;
  const uint8_t* zeros;
};

// row_lo, row_hi: the lane's two rows in the first row tile; rows that do not exist read the last one, their results are not
// written.
template <bool ZEROS, int R, int B, int SPAN>
__device__ __forceinline__ void load_scales(Scales<ZEROS, R, B, SPAN>& h, const Int4Weight& w, const View& v, int tile_row, int kt,
                                            int g, int t) {
  int lo[R], hi[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    lo[i] = min((tile_row + i) * 16 + g, w.N - 1);
    hi[i] = min((tile_row + i) * 16 + g + 8, w.N - 1);
  }
#pragma unroll
  for (int b = 0; b < B; b += SPAN) {
    const int at = int4_group_of(w, min((kt + b) * 64 + t * 16, w.K - 16)) * w.N;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      h.s_lo[b / SPAN][i] = __ldg(v.scales + static_cast<uint32_t>(at + lo[i]));
      h.s_hi[b / SPAN][i] = __ldg(v.scales + static_cast<uint32_t>(at + hi[i]));
      if constexpr (ZEROS) {
        h.z_lo[b / SPAN][i] = __ldg(v.zeros + static_cast<uint32_t>(at + lo[i]));
        h.z_hi[b / SPAN][i] = __ldg(v.zeros + static_cast<uint32_t>(at + hi[i]));
      }
    }
  }
}

// Place of the tile's 16-byte piece t * 8 + g.  Eight lanes of one instruction are one t and all g when they write, two
// neighbouring g and all t when they read; either way the places fall into eight different groups of banks.
__device__ __forceinline__ uint32_t place(int g, int t) { return static_cast<uint32_t>(t * 8 + (g ^ (2 * t))) * 16; }

__device__ __forceinline__ void copy16(uint32_t dst, const uint8_t* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory"); }

// acc += W X^T over step b, whose packed weights lie at `at` (row tiles 512 bytes apart) in shared memory;
// x[j] are the lane's 32 bytes of row 8j + g of X
template <bool BF16, bool ZEROS, int NT, int R, int B, int SPAN, int CH>
__device__ __forceinline__ void multiply(const Scales<ZEROS, R, B, SPAN>& h, int b, bool in, const unsigned char* at,
                                         const uint4 (&x)[NT][2], float (&acc)[R][NT][CH][4]) {
  uint32_t s_lo[R], s_hi[R], o_lo[R], o_hi[R], q[R][4];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const uint4 c = *reinterpret_cast<const uint4*>(at + i * 512);
    q[i][0] = c.x; q[i][1] = c.y; q[i][2] = c.z; q[i][3] = c.w;
    s_lo[i] = in ? h.s_lo[b / SPAN][i] * 0x10001u : 0u;
    s_hi[i] = in ? h.s_hi[b / SPAN][i] * 0x10001u : 0u;
    o_lo[i] = Int4Type<BF16>::offset(ZEROS ? h.z_lo[ZEROS ? b / SPAN : 0][i] & 15 : 8);
    o_hi[i] = int4_offset_hi<BF16>(ZEROS ? h.z_hi[ZEROS ? b / SPAN : 0][i] & 15 : 8);
  }
#pragma unroll
  for (int s = 0; s < 4; ++s)
#pragma unroll
    for (int i = 0; i < R; ++i) {
      uint32_t a[4];
      int4_word<BF16>(q[i][s], o_lo[i], o_hi[i], s_lo[i], s_hi[i], a);
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const uint4& c = x[j][s >> 1];
        mma16816<BF16>(acc[i][j][s % CH], a, (s & 1) ? c.z : c.x, (s & 1) ? c.w : c.y);
      }
    }
}

// The work is chunks of rows of X (one for the dense product; the plan's or one per slot for experts) times the weight's row
// groups (R row tiles each).  The grid is what runs at once; gridDim.x / chunks blocks share a chunk, and there are teams of TW
// warps in a block, team n of the chunk's taking row groups [groups * n / teams, groups * (n + 1) / teams).  The warps of a
// team take the blocks of a row group in turn; their sums meet every RGF row groups.  XS: the rows of X lie in shared memory,
// 16 bytes apart from a multiple of 128, so that the reads of a quarter warp (two rows, four runs of 16 columns) have no bank
// conflicts; else they are read from memory in the loop.
template <bool BF16, bool ZEROS, int MODE, int NT, int R, int B, int SPAN, int SLOTS, int WARPS, int TW, int MIN_BLOCKS, int RGF, bool XS>
__global__ void __launch_bounds__(WARPS * 32, MIN_BLOCKS)
int4_small_kernel(const SmallParams p) {
  using I = Int4Type<BF16>;
  using T = typename I::T;
  constexpr int TEAMS = WARPS / TW;
  constexpr int CH = R * NT == 1 ? 2 : 1;   // chains of accumulators: a matrix instruction waits for the one before it
  constexpr int VALUES = R * NT * 4;        // sums of a lane per row group
  constexpr int BYTES = R * B * 512;
  constexpr int RED = RGF * VALUES * 128;     // per warp
  static_assert(TW > 1, "the sums of a team meet in shared memory");
  extern __shared__ __align__(128) unsigned char smem[];   // rings, sums [team][row group][warp][VALUES][lane], X
  const int warp = (threadIdx.x >> 5) % TW, team = threadIdx.x / (TW * 32), lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const Int4Weight& w = p.w;
  float* red = reinterpret_cast<float*>(smem + WARPS * SLOTS * BYTES) + team * (TW * RED / 4);
  unsigned char* xs = smem + WARPS * (SLOTS * BYTES + RED);
  unsigned char* ring = smem + (team * TW + warp) * (SLOTS * BYTES);
  const uint32_t put = place(lane & 7, lane >> 3), get = place(g, t);
  const int groups = (w.row_tiles() + R - 1) / R, k_tiles = w.k_tiles(), pitch = k_tiles * 128 + 16;
  const bool works = warp * B < k_tiles;                    // the warp has a block of a row group

  grid_release();
  if constexpr (MODE != kDense) grid_wait();               // (the dense product's weights are read before it)
  const int chunks = MODE == kDense ? p.chunks : p.rows.chunks ? *p.rows.n_chunks : p.rows.slots;
  const int per = max(1, static_cast<int>(gridDim.x) / max(1, chunks));    // blocks per chunk
  const int part = blockIdx.x % per, stride = gridDim.x / per;
  for (int chunk = blockIdx.x / per; chunk < chunks; chunk += stride) {
    if (static_cast<int>(blockIdx.x) >= stride * per) break;               // (left over)
    int first = chunk * (8 * NT), count = p.M - first, expert = 0;
    if constexpr (MODE != kDense) {
      if (p.rows.chunks) {
        const int4 c = p.rows.chunks[chunk];
        expert = c.x; first = c.y; count = c.z;
      } else {
        expert = p.rows.ids[chunk]; first = chunk; count = 1;
        if (expert < 0 || expert >= p.rows.E) continue;
      }
    }
    const View v{w.packed + expert * w.expert_bytes() + lane * 16,
                 static_cast<const unsigned short*>(w.scales) + expert * w.expert_scales(),
                 ZEROS ? w.zeros + expert * w.expert_scales() : nullptr};
    const long long teams = static_cast<long long>(per) * TEAMS, me = static_cast<long long>(part) * TEAMS + team;
    const int rg0 = static_cast<int>(groups * me / teams), rg1 = static_cast<int>(groups * (me + 1) / teams);
    const int rows_here = min(count, 8 * NT);

    // the warp's sequence of blocks, and the next one to copy
    int l_rg = works ? rg0 : rg1, l_kt = warp * B;
    auto fill = [&](unsigned char* to) {
      const uint32_t slot = smem_u32(to);
      if (l_rg < rg1) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
          const int tr = R == 1 ? l_rg : min(l_rg * R + i, w.row_tiles() - 1);
          const uint8_t* src = v.packed + (static_cast<size_t>(tr) * k_tiles + l_kt) * 512;
          if (l_kt + B <= k_tiles) {
#pragma unroll
            for (int b = 0; b < B; ++b) copy16(slot + put + (b * R + i) * 512, src + b * 512);
          } else {
#pragma unroll
            for (int b = 0; b < B; ++b)
              if (l_kt + b < k_tiles) copy16(slot + put + (b * R + i) * 512, src + b * 512);
          }
        }
        l_kt += TW * B;
        if (l_kt >= k_tiles) { l_kt = warp * B; ++l_rg; }
      }
      copy_commit();
    };
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) fill(ring + i * BYTES);

    auto x_row = [&](int c) -> const T* {
      long long r = first + c;
      if constexpr (MODE == kGated) r = (p.rows.row_slot ? p.rows.row_slot[r] : r) / p.rows.top_k;
      return static_cast<const T*>(p.x) + r * w.K;
    };
    // columns of the instruction beyond the rows read row 0 again: their results are not written
    const T* xrow[NT];
    const unsigned char* xat[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int c = j * 8 + g < rows_here ? j * 8 + g : 0;
      if constexpr (XS) xat[j] = xs + c * pitch + t * 32;
      else xrow[j] = x_row(c) + t * 16;
    }
    Scales<ZEROS, R, B, SPAN> ahead;
    if (works && rg0 < rg1) load_scales<ZEROS, R, B, SPAN>(ahead, w, v, rg0 * R, warp * B, g, t);
    if constexpr (MODE == kDense) grid_wait();
    if constexpr (XS) {   // columns that fill up the last step are zero
      for (int c = threadIdx.x / 32; c < rows_here; c += WARPS) {
        const uint4* src = reinterpret_cast<const uint4*>(x_row(c));
        for (int i = lane; i < k_tiles * 8; i += 32)
          *reinterpret_cast<uint4*>(xs + c * pitch + i * 16) = i * 8 < w.K ? __ldg(src + i) : make_uint4(0, 0, 0, 0);
      }
      __syncthreads();
    }
    auto load_x = [&](uint4 (&d)[NT][2], int step, bool in) {
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        if constexpr (XS) {
          d[j][0] = *reinterpret_cast<const uint4*>(xat[j] + step * 128);
          d[j][1] = *reinterpret_cast<const uint4*>(xat[j] + step * 128 + 16);
        } else {
          d[j][0] = d[j][1] = make_uint4(0, 0, 0, 0);
          if (in) {
            d[j][0] = __ldg(reinterpret_cast<const uint4*>(xrow[j] + step * 64));
            d[j][1] = __ldg(reinterpret_cast<const uint4*>(xrow[j] + step * 64) + 1);
          }
        }
      }
    };
    // a value of a row group's sums, by its place in the lane's accumulators
    auto write = [&](int rg, int q, float sum) {
      const int c = q & 3, j = (q >> 2) % NT, i = (q >> 2) / NT;
      const int n = (rg * R + i) * 16 + g + (c >> 1) * 8;      // weight row
      const int col = j * 8 + t * 2 + (c & 1);                 // row of the chunk
      if constexpr (MODE == kGated) {
        const float other = __shfl_xor_sync(0xffffffffu, sum, 4);          // rows 2i and 2i + 1 are four lanes apart
        if ((g & 1) == 0 && n + 1 < w.N && col < rows_here)
          static_cast<T*>(p.y)[(static_cast<long long>(first) + col) * (w.N / 2) + n / 2] = I::from_float(silu_mul(sum, other));
      } else if (n < w.N && col < rows_here) {
        const long long row = first + col;
        if constexpr (MODE == kDense) static_cast<T*>(p.y)[row * w.N + n] = I::from_float(sum);
        else static_cast<float*>(p.y)[static_cast<long long>(p.rows.row_slot[row]) * w.N + n] = sum;
      }
    };
    float acc[R][NT][CH][4] = {};
    unsigned char* at = ring;
    for (int rg = rg0; rg < rg1; ++rg) {
      for (int kt = warp * B; kt < k_tiles; kt += TW * B) {
        const Scales<ZEROS, R, B, SPAN> sc = ahead;
        const bool last = kt + TW * B >= k_tiles;              // of the row group
        if (!last || rg + 1 < rg1)
          load_scales<ZEROS, R, B, SPAN>(ahead, w, v, (rg + last) * R, last ? warp * B : kt + TW * B, g, t);
        if ((kt + B) * 64 <= w.K) {
          uint4 x[2][NT][2];
          if constexpr (!XS) load_x(x[0], kt, true);
          copy_wait<SLOTS - 1>();
          __syncwarp();
          if constexpr (XS) load_x(x[0], kt, true);
#pragma unroll
          for (int b = 0; b < B; ++b) {
            if (b + 1 < B) load_x(x[(b + 1) & 1], kt + b + 1, true);
            multiply<BF16, ZEROS, NT, R, B, SPAN, CH>(sc, b, true, at + get + b * (R * 512), x[b & 1], acc);
          }
        } else {   // the row ends inside the block
          copy_wait<SLOTS - 1>();
          __syncwarp();
#pragma unroll
          for (int b = 0; b < B; ++b) {
            if (kt + b < k_tiles) {
              const bool in = (kt + b) * 64 + t * 16 < w.K;
              uint4 x[NT][2];
              load_x(x, kt + b, in);
              multiply<BF16, ZEROS, NT, R, B, SPAN, CH>(sc, b, in, at + get + b * (R * 512), x, acc);
            }
          }
        }
        __syncwarp();                                          // the slot has been read
        fill(at);
        at = at == ring + (SLOTS - 1) * BYTES ? ring : at + BYTES;
      }
      const int n_red = (rg - rg0) % RGF;
      if (works) {
        float* out = red + (n_red * TW + warp) * (VALUES * 32) + lane;
#pragma unroll
        for (int a = 0; a < R; ++a)
#pragma unroll
          for (int b = 0; b < NT; ++b)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const float sum = CH == 2 ? acc[a][b][0][c] + acc[a][b][CH - 1][c] : acc[a][b][0][c];
              out[((a * NT + b) * 4 + c) * 32] = sum;
#pragma unroll
              for (int d = 0; d < CH; ++d) acc[a][b][d][c] = 0.f;
            }
      }
      if (n_red + 1 < RGF && rg + 1 < rg1) continue;
      asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "n"(TW * 32) : "memory");
      const int with_work = min(TW, (k_tiles + B - 1) / B);   // warps that had a block at all
      for (int u = warp; u < (n_red + 1) * VALUES; u += TW) {
        const int r = u / VALUES, q = u % VALUES;
        float sum = 0.f;
        for (int k = 0; k < with_work; ++k) sum += red[((r * TW + k) * VALUES + q) * 32 + lane];
        write(rg - n_red + r, q, sum);
      }
      asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "n"(TW * 32) : "memory");
    }
    if constexpr (XS) __syncthreads();                          // the rows of X may be overwritten
  }
}

// y[token] = sum_j weight_j * H[token * top_k + j] W_{e_j}^T: the K loops of all choices of a token, dealt out to the warps
// one after the other, and the weighted sum in the same reduction.
template <bool BF16, bool ZEROS>
__global__ void __launch_bounds__(kWarps * 32, 1)
int4_small_down_direct_kernel(const SmallParams p) {
  using I = Int4Type<BF16>;
  using T = typename I::T;
  constexpr int B = 2, SLOTS = 2;
  __shared__ __align__(128) unsigned char rings[kWarps][SLOTS][B * 512];
  __shared__ float red[kWarps][2][8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const Int4Weight& w = p.w;
  const int token = blockIdx.y, tile_row = blockIdx.x;
  const int kts = w.k_tiles(), blocks = (kts + B - 1) / B, units = blocks * p.rows.top_k;
  grid_release();
  grid_wait();
  // the warp's share of the blocks of all choices; blocks of dropped choices are passed over
  const int end = static_cast<int>(static_cast<long long>(units) * (warp + 1) / kWarps);
  const int* ids = p.rows.ids + token * p.rows.top_k;
  auto skip = [&](int unit) {   // the first unit from this one on whose choice was not dropped
    while (unit < end) {
      const int e = ids[unit / blocks];
      if (e >= 0 && e < p.rows.E) break;
      unit = (unit / blocks + 1) * blocks;
    }
    return unit;
  };
  unsigned char* ring = &rings[warp][0][0];
  const uint32_t put = place(lane & 7, lane >> 3), get = place(g, t);
  int copy = skip(static_cast<int>(static_cast<long long>(units) * warp / kWarps)), u = copy;
  auto fill = [&](unsigned char* to) {
    if (copy < end) {
      const int kt = (copy % blocks) * B;
      const uint8_t* src = w.packed + ids[copy / blocks] * w.expert_bytes() + (static_cast<size_t>(tile_row) * kts + kt) * 512 + lane * 16;
#pragma unroll
      for (int b = 0; b < B; ++b)
        if (kt + b < kts) copy16(smem_u32(to) + put + b * 512, src + b * 512);
      copy = skip(copy + 1);
    }
    copy_commit();
  };
#pragma unroll
  for (int i = 0; i < SLOTS; ++i) fill(ring + i * (B * 512));
  struct Ahead {
    Scales<ZEROS, 1, B, 1> sc;
    uint4 x[B][1][2];
    float weight;
  };
  auto fetch = [&](Ahead& a, int unit) {
    const int slot = token * p.rows.top_k + unit / blocks, expert = ids[unit / blocks], kt = (unit % blocks) * B;
    const View v{w.packed, static_cast<const unsigned short*>(w.scales) + expert * w.expert_scales(),
                 ZEROS ? w.zeros + expert * w.expert_scales() : nullptr};
    load_scales<ZEROS, 1, B, 1>(a.sc, w, v, tile_row, kt, g, t);
    const T* h = static_cast<const T*>(p.x) + static_cast<long long>(slot) * w.K + t * 16;
#pragma unroll
    for (int b = 0; b < B; ++b) {
      a.x[b][0][0] = a.x[b][0][1] = make_uint4(0, 0, 0, 0);
      if ((kt + b) * 64 + t * 16 < w.K) {
        a.x[b][0][0] = __ldg(reinterpret_cast<const uint4*>(h + (kt + b) * 64));
        a.x[b][0][1] = __ldg(reinterpret_cast<const uint4*>(h + (kt + b) * 64) + 1);
      }
    }
    a.weight = p.rows.weights[slot];
  };
  Ahead now, next;
  if (u < end) fetch(next, u);
  float lo = 0.f, hi = 0.f;
  unsigned char* at = ring;
  while (u < end) {
    now = next;
    const int kt = (u % blocks) * B;
    u = skip(u + 1);
    if (u < end) fetch(next, u);
    float acc[1][1][2][4] = {};
    copy_wait<SLOTS - 1>();
    __syncwarp();
#pragma unroll
    for (int b = 0; b < B; ++b)
      if (kt + b < kts)
        multiply<BF16, ZEROS, 1, 1, B, 1, 2>(now.sc, b, (kt + b) * 64 + t * 16 < w.K, at + get + b * 512, now.x[b], acc);
    __syncwarp();
    fill(at);
    at = at == ring + (SLOTS - 1) * (B * 512) ? ring : at + B * 512;
    lo += now.weight * (acc[0][0][0][0] + acc[0][0][1][0]);
    hi += now.weight * (acc[0][0][0][2] + acc[0][0][1][2]);
  }
  if (t == 0) { red[warp][0][g] = lo; red[warp][1][g] = hi; }
  __syncthreads();
  if (threadIdx.x < 16) {
    const int half = threadIdx.x >> 3, r = threadIdx.x & 7, n = tile_row * 16 + half * 8 + r;
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) v += red[k][half][r];
    if (n < w.N) static_cast<T*>(p.y)[static_cast<long long>(token) * w.N + n] = I::from_float(v);
  }
}

template <bool BF16, bool ZEROS, int MODE, int NT, int R, int B, int SPAN, int SLOTS, int WARPS, int TW, int MIN_BLOCKS, int RGF, bool XS>
int launch_one(const SmallParams& p, int rows, cudaStream_t s) {
  auto kernel = int4_small_kernel<BF16, ZEROS, MODE, NT, R, B, SPAN, SLOTS, WARPS, TW, MIN_BLOCKS, RGF, XS>;
  const long long groups = (p.w.row_tiles() + R - 1) / R;
  const size_t smem = WARPS * (SLOTS * R * B * 512 + RGF * R * NT * 4 * 128) + (XS ? static_cast<size_t>(rows) * (p.w.k_tiles() * 128 + 16) : 0);
  if (smem > kSmallSmem) return VQG_ERR_UNSUPPORTED;
  static SmemOptIn opt_in;
  if (smem > 48 * 1024 && !opt_in.ask(kernel)) return VQG_ERR_LAUNCH;
  // as many blocks as run at once (1 KiB of an SM's shared memory goes with each), or one per row group where there are fewer of those
  const long long slots = static_cast<long long>(sm_count_cached()) * min(MIN_BLOCKS, static_cast<int>(228 * 1024 / (smem + 1024)));
  const int blocks = static_cast<int>(min(slots, groups * p.chunks));
  return cuda_status(launch_ahead(kernel, dim3(blocks), WARPS * 32, smem, s, take_weights_written(s), p));
}

// rows: of a chunk, at most; p.chunks: how many chunks there are, at most
template <int MODE>
int launch_rows(const SmallParams& p, int rows, bool bf16, cudaStream_t s) {
  auto go = [&](auto type, auto zeros) -> int {
    constexpr bool F = decltype(type)::value, Z = decltype(zeros)::value;
    const size_t x = static_cast<size_t>(rows) * (p.w.k_tiles() * 128 + 16);
    if constexpr (MODE == kDense) {
      if (rows <= 8) {
        const bool pairs = p.w.group % 128 == 0;
        // one block of 24 warps per SM: X once per SM
        if (p.w.K >= 64 * 4 * 8 && x + 24 * (2 * 2048 + 1024) <= kSmallSmem)
          return pairs ? launch_one<F, Z, MODE, 1, 1, 4, 2, 2, 24, 8, 1, 2, true>(p, rows, s)
                       : launch_one<F, Z, MODE, 1, 1, 4, 1, 2, 24, 8, 1, 2, true>(p, rows, s);
        if (x <= 32 * 1024) return launch_one<F, Z, MODE, 1, 1, 2, 1, 3, 8, 8, 3, 2, true>(p, rows, s);
        return launch_one<F, Z, MODE, 1, 1, 4, 1, 2, 8, 8, 3, 2, false>(p, rows, s);
      }
      if (rows <= 16) {
        if (x + 16 * (2 * 2048 + 2048) <= kSmallSmem) return launch_one<F, Z, MODE, 2, 2, 2, 1, 2, 16, 8, 1, 1, true>(p, rows, s);
        return launch_one<F, Z, MODE, 2, 2, 2, 1, 3, 8, 8, 2, 1, false>(p, rows, s);
      }
      return launch_one<F, Z, MODE, 4, 2, 2, 1, 2, 8, 8, 2, 1, false>(p, rows, s);
    } else {
      // Experts: short rows and many row groups, so teams of two warps, or of four where there are few slots.
      if (!p.rows.chunks) {
        if (x <= 32 * 1024) return launch_one<F, Z, MODE, 1, 1, 2, 1, 3, 8, 4, 3, 2, true>(p, rows, s);
        return launch_one<F, Z, MODE, 1, 1, 2, 1, 3, 8, 4, 3, 2, false>(p, rows, s);
      }
      if (rows <= 8) {
        // X in shared memory while three blocks fit with it (2432 columns, 8 tokens through 64 experts: two blocks 92 us, three that
        // read X from memory 81)
        if (x <= 35 * 1024) return launch_one<F, Z, MODE, 1, 1, 4, 1, 2, 8, 2, 3, 2, true>(p, rows, s);
        return launch_one<F, Z, MODE, 1, 1, 4, 1, 2, 8, 2, 3, 2, false>(p, rows, s);
      }
      if (x <= 70 * 1024) return launch_one<F, Z, MODE, 2, 1, 4, 1, 2, 8, 2, 2, 1, true>(p, rows, s);
      return launch_one<F, Z, MODE, 2, 1, 4, 1, 2, 8, 2, 2, 1, false>(p, rows, s);
    }
  };
  if (p.w.zeros) return bf16 ? go(std::true_type{}, std::true_type{}) : go(std::false_type{}, std::true_type{});
  return bf16 ? go(std::true_type{}, std::false_type{}) : go(std::false_type{}, std::false_type{});
}

}  // namespace

int launch_int4_small(const Int4Weight& w, const void* x, void* y, int M, bool bf16, cudaStream_t s) {
  SmallParams p{};
  p.w = w; p.x = x; p.y = y; p.M = M;
  const int rows = M <= 8 ? 8 : M <= 16 ? 16 : kInt4SmallRows;
  p.chunks = (M + rows - 1) / rows;
  return launch_rows<kDense>(p, M < rows ? M : rows, bf16, s);
}

int launch_int4_small_gated(const Int4Weight& w, const void* x, void* h, const ExpertRows& rows, int chunk_rows, int max_chunks,
                            bool bf16, cudaStream_t s) {
  SmallParams p{};
  p.w = w; p.x = x; p.y = h; p.rows = rows;
  p.chunks = rows.chunks ? max_chunks : rows.slots;
  return launch_rows<kGated>(p, rows.chunks ? chunk_rows : 1, bf16, s);
}

int launch_int4_small_down(const Int4Weight& w, const void* h, float* part, const ExpertRows& rows, int chunk_rows, int max_chunks,
                           bool bf16, cudaStream_t s) {
  SmallParams p{};
  p.w = w; p.x = h; p.y = part; p.rows = rows;
  p.chunks = max_chunks;
  return launch_rows<kDown>(p, chunk_rows, bf16, s);
}

int launch_int4_small_down_direct(const Int4Weight& w, const void* h, void* y, const ExpertRows& rows, int tokens, bool bf16,
                                  cudaStream_t s) {
  SmallParams p{};
  p.w = w; p.x = h; p.y = y; p.rows = rows;
  const dim3 grid(w.row_tiles(), tokens);
  const bool plain = take_weights_written(s);
  auto go = [&](auto kernel) { return cuda_status(launch_ahead(kernel, grid, kWarps * 32, 0, s, plain, p)); };
  if (w.zeros) return bf16 ? go(int4_small_down_direct_kernel<true, true>) : go(int4_small_down_direct_kernel<false, true>);
  return bf16 ? go(int4_small_down_direct_kernel<true, false>) : go(int4_small_down_direct_kernel<false, false>);
}

}  // namespace vqg
