// Products of a few rows with 4-bit weights (format: int4.cuh): Y[m, n] = sum_k X[m, k] W[n, k], and the two products of
// the experts of a mixture-of-experts layer over the rows that chose them.
//
// A warp owns R row tiles of the weight (16 rows each) and every eighth 64-column tile of K; one 16-byte load per lane and
// tile gives the A fragments of four mma.sync m16n8k16, whose B fragments are 32 consecutive bytes of a row of X per
// lane.  The eight warps' accumulators are summed through shared memory.
#include <type_traits>

#include "int4.cuh"

namespace vqg {
namespace {

constexpr int kWarps = 8;

struct SmallParams {
  Int4Weight w;
  const void* x;
  void* y;
  int M;
  ExpertRows rows;
};

// weights are read once: past L1
__device__ __forceinline__ uint4 ld_stream(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

enum { kDense = 0, kGated = 1, kDown = 2 };

template <bool BF16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// What a lane holds of B neighbouring 64-column steps of R row tiles between load and use: weights, and scales and zero
// points of rows g and g + 8, one for every SPAN steps (2 where a group is a multiple of 128 columns).
template <bool ZEROS, int R, int B, int SPAN>
struct Held {
  static constexpr int S = B / SPAN;
  uint4 w[B][R];
  unsigned short s_lo[S][R], s_hi[S][R];
  uint8_t z_lo[ZEROS ? S : 1][R], z_hi[ZEROS ? S : 1][R];
};

// One expert's weight as a lane sees it.
struct View {
  const uint8_t* packed;          // at the lane's 16 bytes of tile (0, 0)
  const unsigned short* scales;
  const uint8_t* zeros;
};

// Steps kt ... kt + B - 1, all of them whole.  Rows that do not exist read the last one: their results are not written.
template <bool ZEROS, int R, int B, int SPAN>
__device__ __forceinline__ void load_step(Held<ZEROS, R, B, SPAN>& h, int b, const Int4Weight& w, const View& v, int tile_row, int kt,
                                          int g, int t) {
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int tr = R == 1 ? tile_row : min(tile_row + i, w.row_tiles() - 1);
    h.w[b][i] = ld_stream(v.packed + (static_cast<size_t>(tr) * w.k_tiles() + kt) * 512 + b * 512);
    if (b % SPAN == 0) {
      const size_t at = static_cast<size_t>(int4_group_of(w, (kt + b) * 64 + t * 16)) * w.N;
      const int lo = min(tr * 16 + g, w.N - 1), hi = min(tr * 16 + g + 8, w.N - 1);
      h.s_lo[b / SPAN][i] = __ldg(v.scales + at + lo);
      h.s_hi[b / SPAN][i] = __ldg(v.scales + at + hi);
      if constexpr (ZEROS) { h.z_lo[b / SPAN][i] = __ldg(v.zeros + at + lo); h.z_hi[b / SPAN][i] = __ldg(v.zeros + at + hi); }
    }
  }
}

// Any steps: no column beyond K is read, and its weight is zero.
template <bool ZEROS, int R>
__device__ __forceinline__ void load_edge(Held<ZEROS, R, 1, 1>& h, const Int4Weight& w, const View& v, int tile_row, int kt, int g, int t) {
  load_step<ZEROS, R, 1, 1>(h, 0, w, v, tile_row, kt, g, kt * 64 + t * 16 < w.K ? t : 0);
#pragma unroll
  for (int i = 0; i < R; ++i)
    if (kt * 64 + t * 16 >= w.K) h.s_lo[0][i] = h.s_hi[0][i] = 0;
}

// acc += W X^T over step b; x[j] are the lane's 32 bytes of row 8j + g of X
template <bool BF16, bool ZEROS, int NT, int R, int B, int SPAN, int CH>
__device__ __forceinline__ void multiply(const Held<ZEROS, R, B, SPAN>& h, int b, const uint4 (&x)[NT][2], float (&acc)[R][NT][CH][4]) {
  uint32_t s_lo[R], s_hi[R], o_lo[R], o_hi[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    s_lo[i] = h.s_lo[b / SPAN][i] * 0x10001u;
    s_hi[i] = h.s_hi[b / SPAN][i] * 0x10001u;
    o_lo[i] = Int4Type<BF16>::offset(ZEROS ? h.z_lo[ZEROS ? b / SPAN : 0][i] & 15 : 8);
    o_hi[i] = int4_offset_hi<BF16>(ZEROS ? h.z_hi[ZEROS ? b / SPAN : 0][i] & 15 : 8);
  }
#pragma unroll
  for (int s = 0; s < 4; ++s)
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const uint4& q4 = h.w[b][i];
      const uint32_t word = s == 0 ? q4.x : s == 1 ? q4.y : s == 2 ? q4.z : q4.w;
      uint32_t a[4];
      int4_word<BF16>(word, o_lo[i], o_hi[i], s_lo[i], s_hi[i], a);
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const uint4& q = x[j][s >> 1];
        mma16816<BF16>(acc[i][j][s % CH], a, (s & 1) ? q.z : q.x, (s & 1) ? q.w : q.y);
      }
    }
}

__device__ __forceinline__ float silu_mul(float g, float u) { return g / (1.0f + __expf(-g)) * u; }

// Block (bx, by): row groups (R row tiles each) [groups * bx / grid, groups * (bx + 1) / grid) of the weight, rows `by` of X.
// The eight warps take blocks of B steps in turn; a warp walks its blocks of all its row groups as one sequence in which every
// step's registers are loaded again, for the next block, as soon as it is multiplied.
template <bool BF16, bool ZEROS, int MODE, int NT, int R, int B, int SPAN, int MIN_BLOCKS>
__global__ void __launch_bounds__(kWarps * 32, MIN_BLOCKS)
int4_small_kernel(const SmallParams p) {
  using I = Int4Type<BF16>;
  using T = typename I::T;
  constexpr int CH = R * NT == 1 ? 2 : 1;   // chains of accumulators: a matrix instruction waits for the one before it
  constexpr int VALUES = R * NT * 4;        // sums of a lane per row group
  extern __shared__ float red[];            // [row group][warp][VALUES][lane]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const Int4Weight& w = p.w;

  // the rows of this block
  int first = blockIdx.y * (8 * NT), count = p.M - first, expert = 0;
  if constexpr (MODE != kDense) {
    if (p.rows.chunks) {
      if (static_cast<int>(blockIdx.y) >= *p.rows.n_chunks) return;
      const int4 c = p.rows.chunks[blockIdx.y];
      expert = c.x; first = c.y; count = c.z;
    } else {
      expert = p.rows.ids[blockIdx.y]; first = blockIdx.y; count = 1;
      if (expert < 0 || expert >= p.rows.E) return;
    }
  }
  const View v{w.packed + expert * w.expert_bytes() + (t * 8 + g) * 16,
               static_cast<const unsigned short*>(w.scales) + expert * w.expert_scales(),
               ZEROS ? w.zeros + expert * w.expert_scales() : nullptr};
  const int groups = (w.row_tiles() + R - 1) / R;
  const int rg0 = static_cast<int>(static_cast<long long>(groups) * blockIdx.x / gridDim.x);
  const int rg1 = static_cast<int>(static_cast<long long>(groups) * (blockIdx.x + 1) / gridDim.x);
  const int rows_here = min(count, 8 * NT);
  // columns of the instruction beyond the rows read row 0 again: their results are not written
  const T* xrow[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    long long r = first + (j * 8 + g < rows_here ? j * 8 + g : 0);
    if constexpr (MODE == kGated) r = (p.rows.row_slot ? p.rows.row_slot[r] : r) / p.rows.top_k;
    xrow[j] = static_cast<const T*>(p.x) + r * w.K + t * 16;
  }

  const int whole = w.K / (64 * B);                       // blocks of B whole steps
  const int mine = whole > warp ? (whole - warp + kWarps - 1) / kWarps : 0;
  const int total = mine * (rg1 - rg0);
  // the steps behind the whole blocks: one each, dealt out after the blocks
  const int edge0 = whole * B + (warp + kWarps - whole % kWarps) % kWarps;
  int l_rg = rg0, l_kt = warp * B;                        // next block to load
  auto advance = [&]() {
    l_kt += kWarps * B;
    if (l_kt >= whole * B) { l_kt = warp * B; ++l_rg; }
  };
  Held<ZEROS, R, B, SPAN> held;
  if (total > 0) {
#pragma unroll
    for (int b = 0; b < B; ++b) load_step<ZEROS, R, B, SPAN>(held, b, w, v, l_rg * R, l_kt, g, t);
    advance();
  }
  float acc[R][NT][CH][4] = {};
  int kt = warp * B, rg = 0;
  auto finish = [&]() {   // the whole blocks of a row group are done: the steps behind them, and the sums to shared memory
    for (int e = edge0; e < w.k_tiles(); e += kWarps) {
      Held<ZEROS, R, 1, 1> h;
      load_edge<ZEROS, R>(h, w, v, (rg0 + rg) * R, e, g, t);
      uint4 x[NT][2];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        x[j][0] = x[j][1] = make_uint4(0, 0, 0, 0);
        if (e * 64 + t * 16 < w.K) {
          x[j][0] = __ldg(reinterpret_cast<const uint4*>(xrow[j] + e * 64));
          x[j][1] = __ldg(reinterpret_cast<const uint4*>(xrow[j] + e * 64) + 1);
        }
      }
      multiply<BF16, ZEROS, NT, R, 1, 1, CH>(h, 0, x, acc);
    }
    float* out = red + (rg * kWarps + warp) * (VALUES * 32) + lane;
#pragma unroll
    for (int a = 0; a < R; ++a)
#pragma unroll
      for (int b = 0; b < NT; ++b)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          out[((a * NT + b) * 4 + c) * 32] = CH == 2 ? acc[a][b][0][c] + acc[a][b][CH - 1][c] : acc[a][b][0][c];
#pragma unroll
          for (int d = 0; d < CH; ++d) acc[a][b][d][c] = 0.f;
        }
    kt = warp * B;
    ++rg;
  };
  for (int n = 0; n < total; ++n) {
    const bool more = n + 1 < total;
#pragma unroll
    for (int b = 0; b < B; ++b) {
      uint4 x[NT][2];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        x[j][0] = __ldg(reinterpret_cast<const uint4*>(xrow[j] + kt * 64) + b * 8);
        x[j][1] = __ldg(reinterpret_cast<const uint4*>(xrow[j] + kt * 64) + b * 8 + 1);
      }
      multiply<BF16, ZEROS, NT, R, B, SPAN, CH>(held, b, x, acc);
      // (a scale is loaded again with the last step that it serves)
      if (more && SPAN == 1) load_step<ZEROS, R, B, SPAN>(held, b, w, v, l_rg * R, l_kt, g, t);
      if (more && SPAN == 2 && b % 2 == 1) {
        load_step<ZEROS, R, B, SPAN>(held, b - 1, w, v, l_rg * R, l_kt, g, t);
        load_step<ZEROS, R, B, SPAN>(held, b, w, v, l_rg * R, l_kt, g, t);
      }
    }
    if (more) advance();
    kt += kWarps * B;
    if (kt >= whole * B) finish();
  }
  if (mine == 0)
    while (rg < rg1 - rg0) finish();
  __syncthreads();
  for (int u = warp; u < (rg1 - rg0) * VALUES; u += kWarps) {
    const int r = u / VALUES, q = u % VALUES;
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) sum += red[((r * kWarps + k) * VALUES + q) * 32 + lane];
    const int c = q & 3, j = (q >> 2) % NT, i = (q >> 2) / NT;
    const int n = ((rg0 + r) * R + i) * 16 + g + (c >> 1) * 8;    // weight row
    const int col = j * 8 + t * 2 + (c & 1);                       // row of the batch
    if constexpr (MODE == kGated) {
      const float other = __shfl_xor_sync(0xffffffffu, sum, 4);    // rows 2i and 2i + 1 are four lanes apart
      if ((g & 1) == 0 && n + 1 < w.N && col < rows_here)
        static_cast<T*>(p.y)[(static_cast<long long>(first) + col) * (w.N / 2) + n / 2] = I::from_float(silu_mul(sum, other));
    } else if (n < w.N && col < rows_here) {
      const long long row = first + col;
      if constexpr (MODE == kDense) static_cast<T*>(p.y)[row * w.N + n] = I::from_float(sum);
      else static_cast<float*>(p.y)[static_cast<long long>(p.rows.row_slot[row]) * w.N + n] = sum;
    }
  }
}

// y[token] = sum_j weight_j * H[token * top_k + j] W_{e_j}^T: the K loops of all choices of a token, dealt out to the warps
// one after the other, and the weighted sum in the same reduction.
template <bool BF16, bool ZEROS>
__global__ void __launch_bounds__(kWarps * 32, 3)
int4_small_down_direct_kernel(const SmallParams p) {
  using I = Int4Type<BF16>;
  using T = typename I::T;
  constexpr int B = 4;
  __shared__ float red[kWarps][2][8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const Int4Weight& w = p.w;
  const int token = blockIdx.y, tile_row = blockIdx.x;
  const int kts = w.k_tiles(), units = kts * p.rows.top_k;
  float lo = 0.f, hi = 0.f;
  int u = static_cast<int>(static_cast<long long>(units) * warp / kWarps);
  const int end = static_cast<int>(static_cast<long long>(units) * (warp + 1) / kWarps);
  while (u < end) {
    const int j = u / kts, slot = token * p.rows.top_k + j;
    const int kt0 = u - j * kts, kt1 = min(end - j * kts, kts);
    u = j * kts + kt1;
    const int expert = p.rows.ids[slot];
    if (expert < 0 || expert >= p.rows.E) continue;
    const View v{w.packed + expert * w.expert_bytes() + (t * 8 + g) * 16,
                 static_cast<const unsigned short*>(w.scales) + expert * w.expert_scales(),
                 ZEROS ? w.zeros + expert * w.expert_scales() : nullptr};
    const T* h = static_cast<const T*>(p.x) + static_cast<long long>(slot) * w.K + t * 16;
    float acc[1][1][2][4] = {};
    int kt = kt0;
    const int kt_whole = min(kt1, w.K / 64);
    for (; kt + B <= kt_whole; kt += B) {
      Held<ZEROS, 1, B, 1> held;
      uint4 x[B][1][2];
#pragma unroll
      for (int b = 0; b < B; ++b) {
        load_step<ZEROS, 1, B, 1>(held, b, w, v, tile_row, kt, g, t);
        x[b][0][0] = __ldg(reinterpret_cast<const uint4*>(h + kt * 64) + b * 8);
        x[b][0][1] = __ldg(reinterpret_cast<const uint4*>(h + kt * 64) + b * 8 + 1);
      }
#pragma unroll
      for (int b = 0; b < B; ++b) multiply<BF16, ZEROS, 1, 1, B, 1, 2>(held, b, x[b], acc);
    }
    for (; kt < kt1; ++kt) {
      Held<ZEROS, 1, 1, 1> held;
      load_edge<ZEROS, 1>(held, w, v, tile_row, kt, g, t);
      uint4 x[1][2] = {};
      if (kt * 64 + t * 16 < w.K) {
        x[0][0] = __ldg(reinterpret_cast<const uint4*>(h + kt * 64));
        x[0][1] = __ldg(reinterpret_cast<const uint4*>(h + kt * 64) + 1);
      }
      multiply<BF16, ZEROS, 1, 1, 1, 1, 2>(held, 0, x, acc);
    }
    const float weight = p.rows.weights[slot];
    lo += weight * (acc[0][0][0][0] + acc[0][0][1][0]);
    hi += weight * (acc[0][0][0][2] + acc[0][0][1][2]);
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

int sm_count() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms > 0 ? sms : 148;
}

// MAX_GROUPS: row groups whose sums a block has room for in shared memory
template <bool BF16, bool ZEROS, int MODE, int NT, int R, int B, int SPAN, int MIN_BLOCKS, int MAX_GROUPS>
int launch_one(const SmallParams& p, int blocks_y, cudaStream_t s) {
  auto kernel = int4_small_kernel<BF16, ZEROS, MODE, NT, R, B, SPAN, MIN_BLOCKS>;
  const int groups = (p.w.row_tiles() + R - 1) / R;
  // as many blocks as run at once, if that leaves them no more row groups than they have room for; else whole rounds of them
  const int slots = max(1, sm_count() * MIN_BLOCKS / blocks_y);
  const int rounds = (groups + slots * MAX_GROUPS - 1) / (slots * MAX_GROUPS);
  const int blocks = static_cast<int>(min(static_cast<long long>(groups), static_cast<long long>(slots) * rounds));
  const int per_block = (groups + blocks - 1) / blocks;
  const size_t smem = static_cast<size_t>(per_block) * kWarps * R * NT * 4 * 32 * sizeof(float);
  if (smem > 48 * 1024 &&
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) != cudaSuccess)
    return VQG_ERR_LAUNCH;
  kernel<<<dim3(blocks, blocks_y), kWarps * 32, smem, s>>>(p);
  count_launch();
  return cuda_status(cudaGetLastError());
}

template <int MODE>
int launch_rows(const SmallParams& p, int rows, int blocks_y, bool bf16, cudaStream_t s) {
  auto go = [&](auto type, auto zeros) {
    constexpr bool B = decltype(type)::value, Z = decltype(zeros)::value;
    const bool pairs = p.w.group % 128 == 0;
    if (rows <= 8) {
      if (p.w.K < 64 * 4 * kWarps) return launch_one<B, Z, MODE, 1, 1, 2, 1, 3, 8>(p, blocks_y, s);
      return pairs ? launch_one<B, Z, MODE, 1, 1, 4, 2, 3, 8>(p, blocks_y, s) : launch_one<B, Z, MODE, 1, 1, 4, 1, 3, 8>(p, blocks_y, s);
    }
    if (rows <= 16) return launch_one<B, Z, MODE, 2, 2, 2, 1, 2, 4>(p, blocks_y, s);
    return launch_one<B, Z, MODE, 4, 2, 2, 1, 2, 2>(p, blocks_y, s);
  };
  if (p.w.zeros) return bf16 ? go(std::true_type{}, std::true_type{}) : go(std::false_type{}, std::true_type{});
  return bf16 ? go(std::true_type{}, std::false_type{}) : go(std::false_type{}, std::false_type{});
}

}  // namespace

int launch_int4_small(const Int4Weight& w, const void* x, void* y, int M, bool bf16, cudaStream_t s) {
  SmallParams p{};
  p.w = w; p.x = x; p.y = y; p.M = M;
  const int rows = M < kInt4SmallRows ? M : kInt4SmallRows, chunks = (M + rows - 1) / rows;
  if (chunks > 65535) return VQG_ERR_UNSUPPORTED;
  return launch_rows<kDense>(p, rows, chunks, bf16, s);
}

int launch_int4_small_gated(const Int4Weight& w, const void* x, void* h, const ExpertRows& rows, int chunk_rows, int max_chunks,
                            bool bf16, cudaStream_t s) {
  SmallParams p{};
  p.w = w; p.x = x; p.y = h; p.rows = rows;
  if (!rows.chunks) return launch_rows<kGated>(p, 1, rows.slots, bf16, s);
  return launch_rows<kGated>(p, chunk_rows, max_chunks, bf16, s);
}

int launch_int4_small_down(const Int4Weight& w, const void* h, float* part, const ExpertRows& rows, int chunk_rows, int max_chunks,
                           bool bf16, cudaStream_t s) {
  SmallParams p{};
  p.w = w; p.x = h; p.y = part; p.rows = rows;
  return launch_rows<kDown>(p, chunk_rows, max_chunks, bf16, s);
}

int launch_int4_small_down_direct(const Int4Weight& w, const void* h, void* y, const ExpertRows& rows, int tokens, bool bf16,
                                  cudaStream_t s) {
  SmallParams p{};
  p.w = w; p.x = h; p.y = y; p.rows = rows;
  const dim3 grid(w.row_tiles(), tokens);
  auto go = [&](auto kernel) { kernel<<<grid, kWarps * 32, 0, s>>>(p); };
  if (w.zeros) bf16 ? go(int4_small_down_direct_kernel<true, true>) : go(int4_small_down_direct_kernel<false, true>);
  else bf16 ? go(int4_small_down_direct_kernel<true, false>) : go(int4_small_down_direct_kernel<false, false>);
  count_launch();
  return cuda_status(cudaGetLastError());
}

}  // namespace vqg
