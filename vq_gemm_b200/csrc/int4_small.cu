// Products of a few rows with 4-bit weights (format: int4.cuh): Y[m, n] = sum_k X[m, k] W[n, k], and the two products of
// the experts of a mixture-of-experts layer over the rows that chose them.
//
// A warp owns R row tiles of the weight (16 rows each) and every eighth 64-column tile of K; one 16-byte load per lane and
// tile gives the A fragments of four mma.sync m16n8k16, whose B fragments are 32 consecutive bytes of a row of X per
// lane.  The eight warps' accumulators are summed through shared memory.
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

// One lane's share of a weight tile, as loaded.
struct TileRegs {
  uint4 w;
  uint32_t s_lo, s_hi, o_lo, o_hi;   // scales (twice) and offsets of rows g and g + 8
};

// row0 = first row of the tile, kt = tile column, (g, t) = position of the lane
template <bool BF16>
__device__ __forceinline__ TileRegs load_tile(const Int4Weight& w, const uint8_t* packed, const unsigned short* scales,
                                              const uint8_t* zeros, int tile_row, int kt, int g, int t) {
  using I = Int4Type<BF16>;
  TileRegs r;
  r.w = __ldg(reinterpret_cast<const uint4*>(packed + (static_cast<long long>(tile_row) * w.k_tiles() + kt) * 512) + t * 8 + g);
  const int k = kt * 64 + t * 16;
  const int lo = tile_row * 16 + g, hi = lo + 8;
  r.s_lo = r.s_hi = 0;               // a scale of zero where there is no row or column: the fill of the last tiles is not used
  r.o_lo = r.o_hi = I::offset(8);
  if (k < w.K) {
    const long long at = static_cast<long long>(k / w.group) * w.N;
    if (lo < w.N) r.s_lo = __ldg(scales + at + lo) * 0x10001u;
    if (hi < w.N) r.s_hi = __ldg(scales + at + hi) * 0x10001u;
    if (zeros) {
      if (lo < w.N) r.o_lo = I::offset(__ldg(zeros + at + lo) & 15);
      if (hi < w.N) r.o_hi = I::offset(__ldg(zeros + at + hi) & 15);
    }
  }
  return r;
}

template <bool BF16>
__device__ __forceinline__ void decode_word(uint32_t word, const TileRegs& r, uint32_t (&a)[4]) {
  a[0] = int4_pair<BF16, 0, 0>(word, r.o_lo, r.s_lo);
  a[1] = int4_pair<BF16, 1, 0>(word, r.o_hi, r.s_hi);
  a[2] = int4_pair<BF16, 0, 1>(word, r.o_lo, r.s_lo);
  a[3] = int4_pair<BF16, 1, 1>(word, r.o_hi, r.s_hi);
}

__device__ __forceinline__ float silu_mul(float g, float u) { return g / (1.0f + __expf(-g)) * u; }

template <bool BF16, int MODE, int NT, int R>
__global__ void __launch_bounds__(kWarps * 32)
int4_small_kernel(const SmallParams p) {
  using I = Int4Type<BF16>;
  using T = typename I::T;
  extern __shared__ float red[];   // [warp][R * NT * 4][lane]
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
  const uint8_t* packed = w.packed + expert * w.expert_bytes();
  const unsigned short* scales = static_cast<const unsigned short*>(w.scales) + expert * w.expert_scales();
  const uint8_t* zeros = w.zeros ? w.zeros + expert * w.expert_scales() : nullptr;

  for (int done = 0; done < count; done += 8 * NT) {
    if (MODE == kDense && done > 0) break;
    const int rows_here = min(count - done, 8 * NT);
    const T* xrow[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int c = j * 8 + g;
      xrow[j] = nullptr;
      if (c < rows_here) {
        long long r = first + done + c;
        if constexpr (MODE == kGated) r = (p.rows.row_slot ? p.rows.row_slot[r] : r) / p.rows.top_k;
        xrow[j] = static_cast<const T*>(p.x) + r * w.K + t * 16;
      }
    }
    float acc[R][NT][4];
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[i][j][c] = 0.f;

    for (int kt = warp; kt < w.k_tiles(); kt += kWarps) {
      uint32_t b[NT][8];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        uint4 u = make_uint4(0, 0, 0, 0), v = u;
        if (xrow[j] && kt * 64 + t * 16 < w.K) {
          u = __ldg(reinterpret_cast<const uint4*>(xrow[j] + kt * 64));
          v = __ldg(reinterpret_cast<const uint4*>(xrow[j] + kt * 64) + 1);
        }
        b[j][0] = u.x; b[j][1] = u.y; b[j][2] = u.z; b[j][3] = u.w;
        b[j][4] = v.x; b[j][5] = v.y; b[j][6] = v.z; b[j][7] = v.w;
      }
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const int tile_row = blockIdx.x * R + i;
        if (tile_row >= w.row_tiles()) break;
        const TileRegs r = load_tile<BF16>(w, packed, scales, zeros, tile_row, kt, g, t);
        const uint32_t words[4] = {r.w.x, r.w.y, r.w.z, r.w.w};
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          uint32_t a[4];
          decode_word<BF16>(words[s], r, a);
#pragma unroll
          for (int j = 0; j < NT; ++j) mma16816<BF16>(acc[i][j], a, b[j][2 * s], b[j][2 * s + 1]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) red[(warp * (R * NT * 4) + (i * NT + j) * 4 + c) * 32 + lane] = acc[i][j][c];
    __syncthreads();
    for (int u = warp; u < R * NT * 4; u += kWarps) {
      float v = 0.f;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) v += red[(k * (R * NT * 4) + u) * 32 + lane];
      const int c = u & 3, j = (u >> 2) % NT, i = (u >> 2) / NT;
      const int n = (blockIdx.x * R + i) * 16 + g + (c >> 1) * 8;    // weight row
      const int col = j * 8 + t * 2 + (c & 1);                       // row of the batch
      if constexpr (MODE == kGated) {
        const float other = __shfl_xor_sync(0xffffffffu, v, 4);      // rows 2i and 2i + 1 are four lanes apart
        if ((g & 1) == 0 && n + 1 < w.N && col < rows_here)
          static_cast<T*>(p.y)[(static_cast<long long>(first) + done + col) * (w.N / 2) + n / 2] = I::from_float(silu_mul(v, other));
      } else if (n < w.N && col < rows_here) {
        const long long r = first + done + col;
        if constexpr (MODE == kDense) static_cast<T*>(p.y)[r * w.N + n] = I::from_float(v);
        else static_cast<float*>(p.y)[static_cast<long long>(p.rows.row_slot[r]) * w.N + n] = v;
      }
    }
    __syncthreads();
  }
}

// y[token] = sum_j weight_j * H[token * top_k + j] W_{e_j}^T: the K loops of all choices of a token, dealt out to the warps
// one after the other, and the weighted sum in the same reduction.
template <bool BF16>
__global__ void __launch_bounds__(kWarps * 32)
int4_small_down_direct_kernel(const SmallParams p) {
  using I = Int4Type<BF16>;
  using T = typename I::T;
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
    const int stop = min(end, (j + 1) * kts);
    const int expert = p.rows.ids[slot];
    if (expert < 0 || expert >= p.rows.E) { u = stop; continue; }
    const uint8_t* packed = w.packed + expert * w.expert_bytes();
    const unsigned short* scales = static_cast<const unsigned short*>(w.scales) + expert * w.expert_scales();
    const uint8_t* zeros = w.zeros ? w.zeros + expert * w.expert_scales() : nullptr;
    const T* h = static_cast<const T*>(p.x) + static_cast<long long>(slot) * w.K + t * 16;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (; u < stop; ++u) {
      const int kt = u - j * kts;
      uint4 b0 = make_uint4(0, 0, 0, 0), b1 = b0;
      if (g == 0 && kt * 64 + t * 16 < w.K) {
        b0 = __ldg(reinterpret_cast<const uint4*>(h + kt * 64));
        b1 = __ldg(reinterpret_cast<const uint4*>(h + kt * 64) + 1);
      }
      const TileRegs r = load_tile<BF16>(w, packed, scales, zeros, tile_row, kt, g, t);
      const uint32_t words[4] = {r.w.x, r.w.y, r.w.z, r.w.w};
      const uint32_t b[8] = {b0.x, b0.y, b0.z, b0.w, b1.x, b1.y, b1.z, b1.w};
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        uint32_t a[4];
        decode_word<BF16>(words[s], r, a);
        mma16816<BF16>(acc, a, b[2 * s], b[2 * s + 1]);
      }
    }
    const float weight = p.rows.weights[slot];
    lo += weight * acc[0];
    hi += weight * acc[2];
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

template <bool BF16, int MODE, int NT, int R>
int launch_one(const SmallParams& p, int blocks_y, cudaStream_t s) {
  const size_t smem = static_cast<size_t>(kWarps) * R * NT * 4 * 32 * sizeof(float);
  auto kernel = int4_small_kernel<BF16, MODE, NT, R>;
  if (smem > 48 * 1024 &&
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) != cudaSuccess)
    return VQG_ERR_LAUNCH;
  const dim3 grid((p.w.row_tiles() + R - 1) / R, blocks_y);
  kernel<<<grid, kWarps * 32, smem, s>>>(p);
  count_launch();
  return cuda_status(cudaGetLastError());
}

}  // namespace

int launch_int4_small(const Int4Weight& w, const void* x, void* y, int M, bool bf16, cudaStream_t s) {
  SmallParams p{};
  p.w = w; p.x = x; p.y = y; p.M = M;
  if (M <= 8) return bf16 ? launch_one<true, kDense, 1, 1>(p, 1, s) : launch_one<false, kDense, 1, 1>(p, 1, s);
  const int chunks = (M + 31) / 32;
  if (chunks > 65535) return VQG_ERR_UNSUPPORTED;
  return bf16 ? launch_one<true, kDense, 4, 2>(p, chunks, s) : launch_one<false, kDense, 4, 2>(p, chunks, s);
}

int launch_int4_small_gated(const Int4Weight& w, const void* x, void* h, const ExpertRows& rows, int max_chunks, bool bf16,
                            cudaStream_t s) {
  SmallParams p{};
  p.w = w; p.x = x; p.y = h; p.rows = rows;
  if (!rows.chunks) return bf16 ? launch_one<true, kGated, 1, 1>(p, rows.slots, s) : launch_one<false, kGated, 1, 1>(p, rows.slots, s);
  return bf16 ? launch_one<true, kGated, 4, 2>(p, max_chunks, s) : launch_one<false, kGated, 4, 2>(p, max_chunks, s);
}

int launch_int4_small_down(const Int4Weight& w, const void* h, float* part, const ExpertRows& rows, int max_chunks, bool bf16,
                           cudaStream_t s) {
  SmallParams p{};
  p.w = w; p.x = h; p.y = part; p.rows = rows;
  return bf16 ? launch_one<true, kDown, 4, 2>(p, max_chunks, s) : launch_one<false, kDown, 4, 2>(p, max_chunks, s);
}

int launch_int4_small_down_direct(const Int4Weight& w, const void* h, void* y, const ExpertRows& rows, int tokens, bool bf16,
                                  cudaStream_t s) {
  SmallParams p{};
  p.w = w; p.x = h; p.y = y; p.rows = rows;
  const dim3 grid(w.row_tiles(), tokens);
  if (bf16) int4_small_down_direct_kernel<true><<<grid, kWarps * 32, 0, s>>>(p);
  else int4_small_down_direct_kernel<false><<<grid, kWarps * 32, 0, s>>>(p);
  count_launch();
  return cuda_status(cudaGetLastError());
}

}  // namespace vqg
