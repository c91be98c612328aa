// 4-bit weights with group scales: the format, the problem descriptors and the decoding of a packed word.
//
//   W[n, k] = round_T((code[n, k] - zero[k / group, n]) * scale[k / group, n])        T = fp16 or bf16
//
// code and zero are 0 ... 15 (zero is 8 where there are no zero points), scale is of type T.  The difference is a whole
// number of at most five bits and therefore exact in T, so W is the exact product rounded once: every kernel here
// multiplies the same bits that the dequantisation writes.
//
// Storage: tiles of 16 rows x 64 columns, 512 bytes each, [ceil(N/16)][ceil(K/64)] of them.  The byte at
// (((t*8 + g)*4 + s)*2 + e)*2 + q holds column 16t + 4s + 2q + e of row g (low four bits) and of row g + 8 (high four
// bits).  The order is the one the hardware wants: lane t*8 + g of a warp reads its 16 bytes with one load (the warp 512
// contiguous ones); word s of them is the A fragment of one 16x8x16 matrix instruction whose 16 columns are, for thread t
// of a quad, 16t + 4s ... +3 -- a permutation of the tile's columns under which that thread's B fragments are 16
// consecutive values of X; and bits i and i + 16 of a word are neighbouring columns, which one AND turns into a pair.
// Rows and columns that fill up the last tiles hold anything; the kernels do not let them reach a result.
#pragma once

#include <cuda_bf16.h>

#include <atomic>

#include "common.cuh"

namespace vqg {

struct Int4Weight {
  const uint8_t* packed;   // [E][ceil(N/16)][ceil(K/64)][512]
  const void* scales;      // [E][K/group][N] of type T
  const uint8_t* zeros;    // the same shape, or null
  int N, K, group;
  uint32_t group_magic;    // ceil(2^32 / (group / 16)): see group_of()
  __host__ __device__ int row_tiles() const { return (N + 15) / 16; }
  __host__ __device__ int k_tiles() const { return (K + 63) / 64; }
  __host__ __device__ long long expert_bytes() const { return static_cast<long long>(row_tiles()) * k_tiles() * 512; }
  __host__ __device__ long long expert_scales() const { return static_cast<long long>(K / group) * N; }
};

// Rows of a mixture-of-experts batch.  A slot is one (token, choice) pair, slot = token * top_k + choice.  In planned form
// the slots are ordered by expert: `row_slot[r]` is the slot of row r, and chunk c covers rows [chunk.y, chunk.y + chunk.z)
// of expert chunk.x.  In direct form (few slots) row r is slot r and there is no plan.
struct ExpertRows {
  const int* ids;        // [slots] chosen expert of each slot; outside 0 ... E-1: the slot is dropped
  const float* weights;  // [slots]
  const int* row_slot;   // planned form: [slots]
  const int4* chunks;    // planned form
  const int* n_chunks;   // planned form: number of chunks, number of rows
  int E, top_k, slots;
};

int launch_int4_small(const Int4Weight& w, const void* x, void* y, int M, bool bf16, cudaStream_t s);
// H[r, N/2] = SiLU(gate) * up for the rows of a plan (or for every slot in direct form)
int launch_int4_small_gated(const Int4Weight& w, const void* x, void* h, const ExpertRows& rows, int chunk_rows, int max_chunks,
                            bool bf16, cudaStream_t s);
// part[slot, N] fp32 = H[r] * W_e^T for the rows of a plan
int launch_int4_small_down(const Int4Weight& w, const void* h, float* part, const ExpertRows& rows, int chunk_rows, int max_chunks,
                           bool bf16, cudaStream_t s);
// y[token, N] = sum over the token's choices of weight * H[slot] W_e^T, direct form
int launch_int4_small_down_direct(const Int4Weight& w, const void* h, void* y, const ExpertRows& rows, int tokens, bool bf16,
                                  cudaStream_t s);
constexpr int kInt4SmallRows = 32;   // rows of a chunk of the dense product, at most (8, 16 or 32); of an expert's 8 or 16

// Many rows: tcgen05 kernels (int4_tensor.cu).  The dense form deals out K loops evenly if it gets a workspace.
size_t int4_tensor_workspace_bytes();
int launch_int4_tensor(const Int4Weight& w, const void* x, void* y, int M, bool bf16, void* ws, size_t ws_bytes, cudaStream_t s);
// rows of a plan with chunks of up to chunk_rows, kInt4TensorRows at most; x_rows is X in the order of the plan (launch_gather_rows)
int launch_int4_tensor_gated(const Int4Weight& w, const void* x_rows, void* h, const ExpertRows& rows, int chunk_rows, int max_chunks, bool bf16,
                             cudaStream_t s);
int launch_int4_tensor_down(const Int4Weight& w, const void* h, float* part, const ExpertRows& rows, int chunk_rows, int max_chunks, bool bf16,
                            cudaStream_t s);
int launch_gather_rows(const void* x, const ExpertRows& rows, void* out, int cols, cudaStream_t s);
constexpr int kInt4TensorRows = 256;

int launch_int4_dequant(const Int4Weight& w, void* out, int experts, bool bf16, cudaStream_t s);
int launch_int4_quantize(const void* w, uint8_t* packed, void* scales, uint8_t* zeros, int experts, int N, int K, int group,
                         bool bf16, cudaStream_t s);

int launch_route_experts(const void* logits, int logits_type, const float* bias, float* weights, int* ids, int T, int E,
                         int top_k, int scoring, int groups, int top_groups, int group_score, bool renormalize, float scale,
                         cudaStream_t s);
// Orders the slots by expert.  row_slot [slots], chunks [max_chunks], n_chunks [2].
int launch_expert_plan(const int* ids, int slots, int E, int chunk_rows, int* row_slot, int4* chunks, int* n_chunks,
                       cudaStream_t s);
inline int expert_max_chunks(int slots, int E, int chunk_rows) { return slots / chunk_rows + (slots < E ? slots : E); }
// y[t] = sum over j of weights[t, j] * part[t * top_k + j], slots that were dropped left out
int launch_expert_combine(const float* part, const ExpertRows& rows, void* y, int tokens, int cols, bool bf16, cudaStream_t s);

// K up to which 16-column runs are divided by groups with one multiplication: n / d = n * ceil(2^32 / d) >> 32 is exact while
// n * d < 2^32, n and d at most K / 16.
constexpr int kInt4MaxK = 1 << 19;

// Opt-in to large dynamic shared memory, once per kernel and device (a static one per launcher instance): the call to the runtime
// costs a good part of a small launch.
struct SmemOptIn {
  std::atomic<unsigned long long> done{0};
  template <typename Kernel>
  bool ask(Kernel kernel) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0) return false;
    const unsigned long long bit = dev < 64 ? 1ULL << dev : 0;
    if (done.load(std::memory_order_relaxed) & bit) return true;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024) != cudaSuccess) return false;
    done.fetch_or(bit, std::memory_order_relaxed);
    return true;
  }
};

#ifdef __CUDACC__
// Launch with programmatic stream serialisation: the kernel's first instructions may run while the kernel before it on the stream
// finishes.  Every kernel launched this way executes grid_wait() before it reads what an earlier kernel may have written or
// writes anything; only weights, which are constant, are read before it.  `plain`: the weights may have just been written.
template <typename... Params, typename... Args>
cudaError_t launch_ahead(void (*kernel)(Params...), dim3 grid, int threads, size_t smem, cudaStream_t s, bool plain, Args&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = plain ? 0 : 1;
  count_launch();
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
}
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// group of columns k ... k + 15 (k a multiple of 16)
__device__ __forceinline__ int int4_group_of(const Int4Weight& w, int k) {
  return static_cast<int>(__umulhi(static_cast<uint32_t>(k) >> 4, w.group_magic));
}

template <bool BF16>
struct Int4Type;
template <>
struct Int4Type<false> {
  using T = __half;
  static constexpr uint32_t kMagic = 0x64006400u;   // 1024: a code in the low mantissa bits adds its value
  __device__ static uint32_t sub(uint32_t a, uint32_t b) { uint32_t r; asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
  __device__ static uint32_t mul(uint32_t a, uint32_t b) { uint32_t r; asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
  __device__ static uint32_t fma(uint32_t a, uint32_t b, uint32_t c) { uint32_t r; asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c)); return r; }
  __device__ static uint32_t offset(int zero) { return (0x6400u + static_cast<uint32_t>(zero)) * 0x10001u; }   // 1024 + zero, twice
  __device__ static float to_float(T v) { return __half2float(v); }
  __device__ static T from_float(float v) { return __float2half_rn(v); }
};
template <>
struct Int4Type<true> {
  using T = __nv_bfloat16;
  static constexpr uint32_t kMagic = 0x43004300u;   // 128
  __device__ static uint32_t sub(uint32_t a, uint32_t b) { uint32_t r; asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
  __device__ static uint32_t mul(uint32_t a, uint32_t b) { uint32_t r; asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
  __device__ static uint32_t offset(int zero) { return (0x4300u + static_cast<uint32_t>(zero)) * 0x10001u; }
  __device__ static float to_float(T v) { return __bfloat162float(v); }
  __device__ static T from_float(float v) { return __float2bfloat16_rn(v); }
};

// A code becomes a number by the usual conversion of small integers: its bits go into the low mantissa bits of a power of two whose last
// place is one (1024 in fp16, 128 in bf16), and a subtraction of that power, here with the zero point, is exact.
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {   // (a & b) | c
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
// The pair of columns (2q, 2q + 1) of word `w` for row half h: (code - zero) * scale in both halves of the result.
// `off` = Int4Type::offset(zero), `s2` = the scale twice.
template <bool BF16, int H, int Q>
__device__ __forceinline__ uint32_t int4_pair(uint32_t w, uint32_t off, uint32_t s2) {
  using I = Int4Type<BF16>;
  return I::mul(I::sub(and_or(w >> (8 * Q + 4 * H), 0x000f000fu, I::kMagic), off), s2);
}
// The same for row half 1 with the offset that int4_offset_hi gives.  In fp16 the high codes are not shifted down: 1024 + 16 code,
// times 1/16, minus 64 + zero is exact too and saves the shift (bf16 has too few mantissa bits for that).
template <bool BF16, int Q>
__device__ __forceinline__ uint32_t int4_pair_hi(uint32_t w, uint32_t off_hi, uint32_t s2) {
  using I = Int4Type<BF16>;
  if constexpr (BF16) return int4_pair<BF16, 1, Q>(w, off_hi, s2);
  else return I::mul(I::fma(and_or(w >> (8 * Q), 0x00f000f0u, I::kMagic), 0x2c002c00u, off_hi), s2);
}
// The four pairs of a word at once: rows g and g + 8, columns (0, 1) and (2, 3).
template <bool BF16>
__device__ __forceinline__ void int4_word(uint32_t w, uint32_t off_lo, uint32_t off_hi, uint32_t s_lo, uint32_t s_hi, uint32_t (&a)[4]) {
  a[0] = int4_pair<BF16, 0, 0>(w, off_lo, s_lo);
  a[1] = int4_pair_hi<BF16, 0>(w, off_hi, s_hi);
  a[2] = int4_pair<BF16, 0, 1>(w, off_lo, s_lo);
  a[3] = int4_pair_hi<BF16, 1>(w, off_hi, s_hi);
}
// what int4_word wants as the offset of row g + 8: fp16 -(64 + zero) twice (0xd400 = -64, steps of 1/16)
template <bool BF16>
__device__ __forceinline__ uint32_t int4_offset_hi(int zero) {
  return BF16 ? Int4Type<BF16>::offset(zero) : (0xd400u + 16u * static_cast<uint32_t>(zero)) * 0x10001u;
}
// SiLU(g) * u = g / (1 + exp(-g)) * u, with exp(x) = 2^(x log2 e) and both sides of the division times 2^-7: the reciprocal would be zero
// for a divisor above 2^126, which 1 + exp(-g) reaches at g = -87.3; so the result is zero only where g / (1 + exp(-g)) is below the
// normal numbers.  Off by at most 2^-16 of itself (half a step of an argument below 2^8, and 2^-22 each).  Both kernels of the experts'
// layer round it to T, their operand of the second product: beside the result's own rounding that is what separates them from a sum
// in 64 bits (bf16 2.3e-3 of the result instead of 1.7e-3).
__device__ __forceinline__ float silu_mul(float g, float u) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(__fmaf_rn(g, -1.44269504f, -7.f)));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(e + 0.0078125f));
  return (0.0078125f * g) * r * u;
}
template <bool BF16>
__device__ __forceinline__ uint32_t int4_scale2(const void* scales, long long i) {
  return static_cast<uint32_t>(__ldg(static_cast<const unsigned short*>(scales) + i)) * 0x10001u;
}
#endif

}  // namespace vqg
