// Routing to experts, and the bookkeeping of a mixture-of-experts batch.
//
//   p      = softmax(logits) or sigmoid(logits)
//   choice = p + bias (the bias steers the choice and does not enter the weights)
//   groups of consecutive experts: a group's score is the sum of its two largest choices (or the largest); the best
//   top_groups groups stay, equal scores to the lower index
//   ids    = the top_k largest choices among them, in falling order, equal ones to the lower index
//   weight = p[id], divided by their sum if asked, times `scale`
//
// An expert whose logit is -inf or NaN is never chosen; slots for which nothing is left get id -1 and weight 0.
#include "int4.cuh"

namespace vqg {
namespace {

constexpr int kRouteWarps = 4;
constexpr double kNone = -1e300;   // choice of an expert that cannot be chosen

__device__ __forceinline__ float load_logit(const void* p, int type, long long i) {
  if (type == 2) return __ldg(static_cast<const float*>(p) + i);
  const unsigned short v = __ldg(static_cast<const unsigned short*>(p) + i);
  return type == 1 ? __uint_as_float(static_cast<uint32_t>(v) << 16) : __half2float(__ushort_as_half(v));
}

struct RouteParams {
  const void* logits;
  const float* bias;
  float* weights;
  int* ids;
  int T, E, top_k, type, sigmoid, groups, top_groups, group_max, renormalize;
  float scale;
};

// One warp per token; lane l holds experts l, l + 32, ...
template <int EPL>
__global__ void __launch_bounds__(kRouteWarps * 32)
route_kernel(const RouteParams p) {
  __shared__ double s_choice[kRouteWarps][EPL * 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int token = blockIdx.x * kRouteWarps + warp;
  if (token >= p.T) return;
  constexpr unsigned kAll = 0xffffffffu;
  double prob[EPL], choice[EPL];
  double top = kNone;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const int e = lane + 32 * i;
    double x = kNone;
    if (e < p.E) {
      const float l = load_logit(p.logits, p.type, static_cast<long long>(token) * p.E + e);
      if (l > -INFINITY) x = fmin(static_cast<double>(l), 1e200);      // +inf takes all of the softmax
    }
    prob[i] = x;
    top = fmax(top, x);
  }
  for (int d = 16; d; d >>= 1) top = fmax(top, __shfl_xor_sync(kAll, top, d));
  if (p.sigmoid) {
#pragma unroll
    for (int i = 0; i < EPL; ++i) prob[i] = prob[i] > kNone ? 1.0 / (1.0 + exp(-prob[i])) : -1.0;
  } else {
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      prob[i] = prob[i] > kNone ? exp(prob[i] - top) : -1.0;
      sum += fmax(prob[i], 0.0);
    }
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(kAll, sum, d);
#pragma unroll
    for (int i = 0; i < EPL; ++i) prob[i] = prob[i] >= 0.0 ? prob[i] / sum : -1.0;
  }
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const int e = lane + 32 * i;
    choice[i] = prob[i] < 0.0 ? kNone : p.bias ? prob[i] + static_cast<double>(__ldg(p.bias + e)) : prob[i];
  }
  if (p.groups > 1) {
    const int size = p.E / p.groups;
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (lane + 32 * i < p.E) s_choice[warp][lane + 32 * i] = choice[i];
    __syncwarp();
    double score = kNone;
    if (lane < p.groups) {
      double first = kNone, second = kNone;
      for (int i = 0; i < size; ++i) {
        const double c = s_choice[warp][lane * size + i];
        if (c > first) { second = first; first = c; }
        else if (c > second) second = c;
      }
      score = p.group_max || second <= kNone ? first : first + second;
    }
    int better = 0;
    for (int j = 0; j < p.groups; ++j) {
      const double other = __shfl_sync(kAll, score, j);
      better += other > score || (other == score && j < lane);
    }
    const unsigned kept = __ballot_sync(kAll, lane < p.groups && better < p.top_groups);
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const int e = lane + 32 * i;
      if (e < p.E && !(kept >> (e / size) & 1u)) choice[i] = kNone;
    }
  }
  double chosen = 0.0, total = 0.0;   // lane j keeps slot j's weight
  int id = -1;
  for (int j = 0; j < p.top_k; ++j) {
    double best = kNone, bp = 0.0;
    int at = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (choice[i] > best) { best = choice[i]; bp = prob[i]; at = lane + 32 * i; }
    for (int d = 16; d; d >>= 1) {
      const double ob = __shfl_xor_sync(kAll, best, d), op = __shfl_xor_sync(kAll, bp, d);
      const int oa = __shfl_xor_sync(kAll, at, d);
      if (ob > best || (ob == best && oa < at)) { best = ob; bp = op; at = oa; }
    }
    if (best <= kNone) break;
    if (lane == j) { chosen = bp; id = at; }
    total += bp;
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (at == lane + 32 * i) choice[i] = kNone;
  }
  if (lane < p.top_k) {
    if (p.renormalize) chosen = total > 0.0 ? chosen / total : 0.0;
    const long long o = static_cast<long long>(token) * p.top_k + lane;
    p.weights[o] = static_cast<float>(chosen * static_cast<double>(p.scale));
    p.ids[o] = id;
  }
}

// Slots by expert, one block: counts in shared memory, an exclusive scan, places by atomics.  The order of an expert's rows
// depends on the atomics; no result does, every row of a product being computed on its own.
constexpr int kPlanThreads = 1024;
__global__ void __launch_bounds__(kPlanThreads)
expert_plan_kernel(const int* __restrict__ ids, int slots, int E, int chunk_rows, int* __restrict__ row_slot,
                   int4* __restrict__ chunks, int* __restrict__ n_chunks) {
  extern __shared__ int sm[];   // count [E], first row [E], first chunk [E]
  int* count = sm;
  int* row0 = sm + E;
  int* chunk0 = sm + 2 * E;
  for (int e = threadIdx.x; e < E; e += kPlanThreads) count[e] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < slots; i += kPlanThreads) {
    const int e = ids[i];
    if (e >= 0 && e < E) atomicAdd(count + e, 1);
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    int r = 0, c = 0;
    for (int e = 0; e < E; ++e) {
      row0[e] = r; chunk0[e] = c;
      r += count[e]; c += (count[e] + chunk_rows - 1) / chunk_rows;
    }
    n_chunks[0] = c;
    n_chunks[1] = r;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < E; e += kPlanThreads)
    for (int i = 0, c = chunk0[e]; i < count[e]; i += chunk_rows, ++c)
      chunks[c] = make_int4(e, row0[e] + i, min(chunk_rows, count[e] - i), 0);
  __syncthreads();
  for (int i = threadIdx.x; i < slots; i += kPlanThreads) {
    const int e = ids[i];
    if (e >= 0 && e < E) row_slot[atomicAdd(row0 + e, 1)] = i;
  }
}

template <bool BF16>
__global__ void __launch_bounds__(256)
expert_combine_kernel(const float* __restrict__ part, const ExpertRows rows, void* __restrict__ y, int cols) {
  using I = Int4Type<BF16>;
  const int token = blockIdx.x;
  for (int c = threadIdx.x * 4; c < cols; c += 256 * 4) {   // cols is a multiple of 4
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int j = 0; j < rows.top_k; ++j) {
      const int slot = token * rows.top_k + j, e = rows.ids[slot];
      if (e < 0 || e >= rows.E) continue;
      const float weight = rows.weights[slot];
      const float4 v = __ldcs(reinterpret_cast<const float4*>(part + static_cast<long long>(slot) * cols + c));
      sum.x += weight * v.x; sum.y += weight * v.y; sum.z += weight * v.z; sum.w += weight * v.w;
    }
    typename I::T out[4] = {I::from_float(sum.x), I::from_float(sum.y), I::from_float(sum.z), I::from_float(sum.w)};
    *reinterpret_cast<uint2*>(static_cast<typename I::T*>(y) + static_cast<long long>(token) * cols + c) = *reinterpret_cast<uint2*>(out);
  }
}

}  // namespace

int launch_route_experts(const void* logits, int logits_type, const float* bias, float* weights, int* ids, int T, int E,
                         int top_k, int scoring, int groups, int top_groups, int group_score, bool renormalize, float scale,
                         cudaStream_t s) {
  RouteParams p{logits, bias, weights, ids, T, E, top_k, logits_type, scoring, groups, top_groups, group_score,
                renormalize ? 1 : 0, scale};
  const int blocks = (T + kRouteWarps - 1) / kRouteWarps;
  auto go = [&](auto kernel) {
    kernel<<<blocks, kRouteWarps * 32, 0, s>>>(p);
    count_launch();
    return cuda_status(cudaGetLastError());
  };
  if (E <= 64) return go(route_kernel<2>);
  if (E <= 128) return go(route_kernel<4>);
  if (E <= 256) return go(route_kernel<8>);
  if (E <= 512) return go(route_kernel<16>);
  return VQG_ERR_UNSUPPORTED;
}

int launch_expert_plan(const int* ids, int slots, int E, int chunk_rows, int* row_slot, int4* chunks, int* n_chunks,
                       cudaStream_t s) {
  expert_plan_kernel<<<1, kPlanThreads, static_cast<size_t>(E) * 3 * sizeof(int), s>>>(ids, slots, E, chunk_rows, row_slot,
                                                                                       chunks, n_chunks);
  count_launch();
  return cuda_status(cudaGetLastError());
}

int launch_expert_combine(const float* part, const ExpertRows& rows, void* y, int tokens, int cols, bool bf16, cudaStream_t s) {
  if (bf16) expert_combine_kernel<true><<<tokens, 256, 0, s>>>(part, rows, y, cols);
  else expert_combine_kernel<false><<<tokens, 256, 0, s>>>(part, rows, y, cols);
  count_launch();
  return cuda_status(cudaGetLastError());
}

}  // namespace vqg
