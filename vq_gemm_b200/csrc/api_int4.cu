// extern "C" entry points of the 4-bit products, their quantiser and the experts' layer: argument checks, routes, scratch.
#include <atomic>

#include "int4.cuh"

using namespace vqg;

namespace vqg {
int sm_count_cached() {
  static std::atomic<int> known[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  int n = known[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1) return 148;
    known[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}
}  // namespace vqg

namespace {

bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// A group is 32 columns, a multiple of 64, or the whole row; a row is a whole number of groups.
bool group_ok(int K, int group) { return K % 32 == 0 && group > 0 && K % group == 0 && (group == 32 || group % 64 == 0 || group == K); }

// Rows of X or of a weight, at most: row numbers are 32 bits and are rounded up to whole tiles of up to 256.
constexpr int kMaxRows = 0x7fffffff - 511;

int check_weight(const void* packed, const void* scales, const void* zeros, int experts, int N, int K, int group, int dtype) {
  if (experts < 0 || N < 0 || K < 0 || (dtype != 0 && dtype != 1)) return VQG_ERR_BAD_ARG;
  if (experts == 0 || N == 0 || K == 0) return VQG_OK;
  if (!group_ok(K, group) || K > kInt4MaxK || N > kMaxRows) return VQG_ERR_UNSUPPORTED;
  if (static_cast<long long>(K / group) * N > 0x7fffffffLL) return VQG_ERR_UNSUPPORTED;   // 32-bit positions of scales
  if (!packed || !scales || !aligned(packed, 16) || !aligned(scales, 2)) return VQG_ERR_BAD_ARG;
  (void)zeros;   // bytes: any address
  return VQG_OK;
}

Int4Weight weight(const void* packed, const void* scales, const void* zeros, int N, int K, int group) {
  Int4Weight w{};
  w.packed = static_cast<const uint8_t*>(packed);
  w.scales = scales;
  w.zeros = static_cast<const uint8_t*>(zeros);
  w.N = N; w.K = K; w.group = group;
  w.group_magic = static_cast<uint32_t>(((1ULL << 32) + group / 16 - 1) / (group / 16));
  return w;
}

size_t up(size_t n) { return (n + 255) / 256 * 256; }

// Whether a batch is worked on slot by slot, without ordering it by expert: two launches instead of four or five, but an expert that
// several slots chose is read and decoded for each of them.  Worth it while what an even routing repeats costs less than the plan:
// a slot some 1.5 million weights' time beside its own, the plan 26 million's.  Slot by slot and planned, us: 64 experts of 2048 x
// 1024, 8 a token, 1 token 18 and 27, 2 tokens 30 and 38, 3 tokens 43 and 41, 4 tokens 56 and 51; 8 experts, 2 a token, of 1024 x 512
// 4 tokens 10.5 and 14, 8 tokens 17 and 14.5, of 4096 x 4096 2 tokens 57 and 64, 4 tokens 99 and 73, 16 tokens 374 and 90, of 4096 x
// 14336 1 token 88 and 103, 2 tokens 168 and 172, 16 tokens 1213 and 244.
bool experts_direct(int T, int top_k, int E, int hidden, int inner) {
  if (static_cast<long long>(T) * top_k > 32) return false;
  const double share = top_k < E ? static_cast<double>(top_k) / E : 1.0;
  double missed = 1.0;                                         // by all tokens
  for (int t = 0; t < T; ++t) missed *= 1.0 - share;
  const double repeats = T * top_k - E * (1.0 - missed);
  return repeats * (3.0 * hidden * inner + 1.5e6) <= 26e6;
}

// The dense product goes to the tensor-memory kernel above 32 rows, above 16 for weights of 2^24 places or more, above 8 for more
// than 3 * 2^24.  Few-rows kernel and the other: 32 rows of 1024 x 1024 3.6 and 6.8 us, of 4096 x 4096 12.0 and 11.1, of 6144 x
// 4096 15.3 and 12.5; 16 rows of 6144 x 4096 10.0 and 12.4, of 11008 x 4096 14.0 and 15.3, of 4096 x 14336 24.3 and 17.2, of
// 28672 x 8192 54 and 45 (and 8 rows of it 37 and 44).
bool gemm_on_tensor(int M, int N, int K) {
  const long long places = static_cast<long long>(N) * K;
  return M > 32 || (M > 16 && places >= (1 << 24)) || (M > 8 && places > 3 * (1 << 24));
}
// Rows per expert, on average, from which the experts' products do: 4 where the down weights have more than 2^25 places in all, else
// 11.  Both again: 64 experts of 2048 x 1024 at 4 rows 98 and 96 us, at 6 109 and 97, at 10 121 and 98; 8 of 4096 x 14336 at 5 322
// and 263; 8 of 1024 x 512 at 9 17.5 and 19.5, at 11 19.7 and 19.9.
bool experts_on_tensor(long long slots, int E, int hidden, int inner) {
  return slots >= (static_cast<long long>(E) * hidden * inner > (1 << 25) ? 4LL : 11LL) * E;
}
// Rows of a chunk of an expert's rows: what most experts have, so that few read their weights twice.  (128 is the tensor-memory
// kernel's short shape: 768 tokens through 64 experts, 96 rows each, 138 us with it and 163 without.)
int expert_chunk_rows(long long slots, int E, bool tensor) {
  if (tensor) return slots <= 96LL * E ? 128 : kInt4TensorRows;
  return slots <= 5LL * E ? 8 : 16;
}

struct ExpertScratch {
  size_t h, rows, part, row_slot, chunks, n_chunks, total;
};
ExpertScratch expert_scratch(int T, int top_k, int E, int hidden, int inner) {
  ExpertScratch a{};
  const size_t slots = static_cast<size_t>(T) * top_k;
  a.h = 0;
  a.rows = a.h + up(slots * inner * 2);
  const bool tensor = experts_on_tensor(slots, E, hidden, inner), planned = !experts_direct(T, top_k, E, hidden, inner);
  a.part = a.rows + (tensor && planned ? up(slots * hidden * 2) : 0);
  a.row_slot = a.part + (planned ? up(slots * hidden * 4) : 0);
  a.chunks = a.row_slot + up(slots * 4);
  a.n_chunks = a.chunks + up(static_cast<size_t>(expert_max_chunks(static_cast<int>(slots), E, expert_chunk_rows(slots, E, tensor))) * sizeof(int4));
  a.total = a.n_chunks + 256;
  return a;
}

}  // namespace

extern "C" {

size_t vqg_int4_workspace_bytes(int M, int N, int K) {
  return N > 0 && K > 0 && gemm_on_tensor(M, N, K) ? int4_tensor_workspace_bytes() : 0;
}

int vqg_int4_gemm(const void* x, const void* packed, const void* scales, const void* zeros, void* y, int M, int N, int K,
                  int group, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  if (M < 0) return VQG_ERR_BAD_ARG;
  const int st = check_weight(packed, scales, zeros, 1, N, K, group, dtype);
  if (st != VQG_OK) return st;
  if (M == 0 || N == 0) return VQG_OK;
  if (M > kMaxRows) return VQG_ERR_UNSUPPORTED;
  if (!y || !aligned(y, 16)) return VQG_ERR_BAD_ARG;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (K == 0) return cuda_status(cudaMemsetAsync(y, 0, static_cast<size_t>(M) * N * 2, s));
  if (!x || !aligned(x, 16)) return VQG_ERR_BAD_ARG;
  if (ensure_status_word() != cudaSuccess) return VQG_ERR_NO_DEVICE;
  const Int4Weight w = weight(packed, scales, zeros, N, K, group);
  if (gemm_on_tensor(M, N, K)) {
    if (!workspace || workspace_bytes < vqg_int4_workspace_bytes(M, N, K) || !aligned(workspace, 256)) return VQG_ERR_WORKSPACE;
    return launch_int4_tensor(w, x, y, M, dtype == 1, workspace, workspace_bytes, s);
  }
  return launch_int4_small(w, x, y, M, dtype == 1, s);
}

int vqg_int4_dequant(const void* packed, const void* scales, const void* zeros, void* w_out, int experts, int N, int K,
                     int group, int dtype, void* stream) {
  const int st = check_weight(packed, scales, zeros, experts, N, K, group, dtype);
  if (st != VQG_OK) return st;
  if (experts == 0 || N == 0 || K == 0) return VQG_OK;
  if (experts > 65535) return VQG_ERR_UNSUPPORTED;
  if (!w_out || !aligned(w_out, 16)) return VQG_ERR_BAD_ARG;
  if (ensure_status_word() != cudaSuccess) return VQG_ERR_NO_DEVICE;
  return launch_int4_dequant(weight(packed, scales, zeros, N, K, group), w_out, experts, dtype == 1, static_cast<cudaStream_t>(stream));
}

int vqg_int4_quantize(const void* w, void* packed_out, void* scales_out, void* zeros_out, int experts, int N, int K, int group,
                      int dtype, void* stream) {
  const int st = check_weight(packed_out, scales_out, zeros_out, experts, N, K, group, dtype);
  if (st != VQG_OK) return st;
  if (experts == 0 || N == 0 || K == 0) return VQG_OK;
  if (experts > 65535) return VQG_ERR_UNSUPPORTED;
  if (!w || !aligned(w, 16)) return VQG_ERR_BAD_ARG;
  if (ensure_status_word() != cudaSuccess) return VQG_ERR_NO_DEVICE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  note_weights_written(s);
  return launch_int4_quantize(w, static_cast<uint8_t*>(packed_out), scales_out, static_cast<uint8_t*>(zeros_out), experts, N, K,
                              group, dtype == 1, s);
}

int vqg_route_experts(const void* logits, const void* bias, void* weights_out, void* experts_out, int T, int E, int top_k,
                      int scoring, int groups, int top_groups, int group_score, int renormalize, float scale, int logits_dtype,
                      void* stream) {
  if (T < 0 || E < 1 || top_k < 1 || top_k > E) return VQG_ERR_BAD_ARG;
  if (scoring < 0 || scoring > 1 || group_score < 0 || group_score > 1 || logits_dtype < 0 || logits_dtype > 2) return VQG_ERR_BAD_ARG;
  if (groups < 1 || E % groups != 0 || top_groups < 1 || top_groups > groups) return VQG_ERR_BAD_ARG;
  if (E > 512 || top_k > 32 || groups > 32 || T > kMaxRows) return VQG_ERR_UNSUPPORTED;
  if (T == 0) return VQG_OK;
  if (!logits || !weights_out || !experts_out || !aligned(logits, logits_dtype == 2 ? 4 : 2) || !aligned(bias, 4) ||
      !aligned(weights_out, 4) || !aligned(experts_out, 4))
    return VQG_ERR_BAD_ARG;
  if (ensure_status_word() != cudaSuccess) return VQG_ERR_NO_DEVICE;
  return launch_route_experts(logits, logits_dtype, static_cast<const float*>(bias), static_cast<float*>(weights_out),
                              static_cast<int*>(experts_out), T, E, top_k, scoring, groups, top_groups, group_score,
                              renormalize != 0, scale, static_cast<cudaStream_t>(stream));
}

size_t vqg_int4_experts_workspace_bytes(int T, int top_k, int E, int hidden, int inner) {
  if (T <= 0 || top_k <= 0 || E <= 0 || hidden <= 0 || inner <= 0) return 0;
  return expert_scratch(T, top_k, E, hidden, inner).total;
}

int vqg_int4_experts(const void* x, const void* experts, const void* weights, const void* up_packed, const void* up_scales,
                     const void* up_zeros, const void* down_packed, const void* down_scales, const void* down_zeros, void* y,
                     int T, int top_k, int E, int hidden, int inner, int up_group, int down_group, int dtype, void* workspace,
                     size_t workspace_bytes, void* stream) {
  if (T < 0 || top_k < 1 || E < 1 || hidden < 1 || inner < 1 || inner > 0x3fffffff) return VQG_ERR_BAD_ARG;
  int st = check_weight(up_packed, up_scales, up_zeros, E, 2 * inner, hidden, up_group, dtype);
  if (st == VQG_OK) st = check_weight(down_packed, down_scales, down_zeros, E, hidden, inner, down_group, dtype);
  if (st != VQG_OK) return st;
  if (T == 0) return VQG_OK;
  if (E > 512 || static_cast<long long>(T) * top_k > 0x3fffffffLL) return VQG_ERR_UNSUPPORTED;
  if (!x || !experts || !weights || !y || !aligned(x, 16) || !aligned(y, 16) || !aligned(experts, 4) || !aligned(weights, 4))
    return VQG_ERR_BAD_ARG;
  const ExpertScratch at = expert_scratch(T, top_k, E, hidden, inner);
  if (!workspace || workspace_bytes < at.total || !aligned(workspace, 256)) return VQG_ERR_WORKSPACE;
  if (ensure_status_word() != cudaSuccess) return VQG_ERR_NO_DEVICE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool bf16 = dtype == 1;
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  const Int4Weight gu = weight(up_packed, up_scales, up_zeros, 2 * inner, hidden, up_group);
  const Int4Weight dn = weight(down_packed, down_scales, down_zeros, hidden, inner, down_group);
  ExpertRows rows{};
  rows.ids = static_cast<const int*>(experts);
  rows.weights = static_cast<const float*>(weights);
  rows.E = E; rows.top_k = top_k; rows.slots = T * top_k;
  void* h = ws + at.h;
  if (experts_direct(T, top_k, E, hidden, inner)) {
    st = launch_int4_small_gated(gu, x, h, rows, 1, 0, bf16, s);
    if (st != VQG_OK) return st;
    return launch_int4_small_down_direct(dn, h, y, rows, T, bf16, s);
  }
  float* part = reinterpret_cast<float*>(ws + at.part);
  int* row_slot = reinterpret_cast<int*>(ws + at.row_slot);
  int4* chunks = reinterpret_cast<int4*>(ws + at.chunks);
  int* n_chunks = reinterpret_cast<int*>(ws + at.n_chunks);
  const bool tensor = experts_on_tensor(rows.slots, E, hidden, inner);
  const int chunk = expert_chunk_rows(rows.slots, E, tensor), most = expert_max_chunks(rows.slots, E, chunk);
  st = launch_expert_plan(rows.ids, rows.slots, E, chunk, row_slot, chunks, n_chunks, s);
  if (st != VQG_OK) return st;
  rows.row_slot = row_slot; rows.chunks = chunks; rows.n_chunks = n_chunks;
  if (tensor) {
    st = launch_gather_rows(x, rows, ws + at.rows, hidden, s);
    if (st == VQG_OK) st = launch_int4_tensor_gated(gu, ws + at.rows, h, rows, chunk, most, bf16, s);
    if (st == VQG_OK) st = launch_int4_tensor_down(dn, h, part, rows, chunk, most, bf16, s);
  } else {
    st = launch_int4_small_gated(gu, x, h, rows, chunk, most, bf16, s);
    if (st == VQG_OK) st = launch_int4_small_down(dn, h, part, rows, chunk, most, bf16, s);
  }
  if (st == VQG_OK) st = launch_expert_combine(part, rows, y, T, hidden, bf16, s);
  return st;
}

}  // extern "C"
