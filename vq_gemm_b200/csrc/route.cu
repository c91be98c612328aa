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
constexpr unsigned kAll = 0xffffffffu;
constexpr double kNone = -1e300;   // choice of an expert that cannot be chosen, in 64 bits; -inf in 32

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

__device__ __forceinline__ float warp_max(float v) {
  float r;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(kAll, v, d);
  return v;
}

// The definition in 64 bits, for the rows whose order 32 bits do not settle.  One warp; lane l holds experts l, l + 32, ...;
// `s_choice` has room for E values.
template <int EPL>
__device__ __noinline__ void route_row_64(const RouteParams& p, int token, double* s_choice) {
  const int lane = threadIdx.x & 31;
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
      if (lane + 32 * i < p.E) s_choice[lane + 32 * i] = choice[i];
    __syncwarp();
    double score = kNone;
    if (lane < p.groups) {
      double first = kNone, second = kNone;
      for (int i = 0; i < size; ++i) {
        const double c = s_choice[lane * size + i];
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

// One warp per token, in 32 bits, with a proof that 64 would choose the same: choices that follow one another in the order (and
// the last kept and first dropped group) must be further apart than the arithmetic below can be wrong; rows where they are
// not are done again in 64 bits.  Without bias and groups the order is that of the logits themselves, which are compared
// exactly.  A row of 256 experts costs some 500 warp instructions, most of them in the top_k rounds (a maximum over the warp,
// the lowest index that has it, a new maximum for the lane that lost it): the kernel is bound by issue, not by its bytes.
template <int EPL>
__global__ void __launch_bounds__(kRouteWarps * 32)
route_kernel(const RouteParams p) {
  __shared__ double s_choice[kRouteWarps][EPL * 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int token = blockIdx.x * kRouteWarps + warp;
  if (token >= p.T) return;
  const bool plain = !p.bias && p.groups == 1;
  float choice[EPL], prob[EPL];   // prob: exp(logit - top) or the sigmoid
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const int e = lane + 32 * i;
    float l = -INFINITY;
    if (e < p.E) l = fmaxf(load_logit(p.logits, p.type, static_cast<long long>(token) * p.E + e), -INFINITY);   // NaN: -inf
    choice[i] = l;
    top = fmaxf(top, l);
  }
  top = warp_max(top);
  bool sure = top < INFINITY;
  float inverse = 1.f;            // of the softmax's sum
  if (p.sigmoid) {
#pragma unroll
    for (int i = 0; i < EPL; ++i) prob[i] = 1.f / (1.f + expf(-choice[i]));
  } else {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      prob[i] = choice[i] > -INFINITY ? expf(choice[i] - top) : 0.f;
      sum += prob[i];
    }
    sum = warp_sum(sum);
    inverse = sum > 0.f ? 1.f / sum : 0.f;
  }
  // 32-bit errors, relative to p: the exponential 2^-22, its sum with one and the division 2^-24 each; in the softmax also the
  // exponent's difference (at most 2^-25 of it, times what is left of p) and a sum of at most 16 + 5 roundings.  Adding the bias
  // rounds once more.  `slack` is twice what that comes to, relative to what goes in.
  const float slack = p.sigmoid ? 1.f / (1 << 20) : 1.f / (1 << 18);
  if (!plain) {
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const int e = lane + 32 * i;
      if (choice[i] > -INFINITY) {
        prob[i] *= inverse;
        choice[i] = p.bias ? fmaxf(prob[i] + __ldg(p.bias + e), -INFINITY) : prob[i];
      }
    }
    inverse = 1.f;
  }
  if (p.groups > 1) {
    const int size = p.E / p.groups;
    float* s = reinterpret_cast<float*>(s_choice[warp]);
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (lane + 32 * i < p.E) s[lane + 32 * i] = choice[i];
    __syncwarp();
    // 32 / 2^n lanes per group, 2^n >= groups; each starts at another place, so that the groups' reads spread over the banks
    const int shift = 32 - __clz(p.groups - 1), per = 32 >> shift;   // lanes per group
    const int group = lane >> (5 - shift), sub = lane & (per - 1);
    float first = -INFINITY, second = -INFINITY;
    if (group < p.groups) {
      const int n = (size - sub + per - 1) / per;
      int at = n > 0 ? group % n : 0;
      for (int i = 0; i < n; ++i) {
        const float c = s[group * size + sub + per * at];
        if (++at == n) at = 0;
        second = fmaxf(second, fminf(first, c));
        first = fmaxf(first, c);
      }
    }
    for (int d = 1; d < per; d <<= 1) {
      const float of = __shfl_xor_sync(kAll, first, d), os = __shfl_xor_sync(kAll, second, d);
      second = fmaxf(fminf(first, of), fmaxf(second, os));
      first = fmaxf(first, of);
    }
    const bool mine = group < p.groups && sub == 0;
    const float score = p.group_max || second == -INFINITY ? first : first + second;
    const float size_of = p.bias ? 1.f + fabsf(first) + fabsf(second > -INFINITY ? second : 0.f) : first + fmaxf(second, 0.f);
    int better = 0;
    for (int j = 0; j < p.groups; ++j) {
      const float other = __shfl_sync(kAll, score, j << (5 - shift));
      better += other > score || (other == score && j < group);
    }
    const bool keep = mine && better < p.top_groups;
    // (p is at most 1, and without bias it is the choice)
    const float low = keep && score > -INFINITY ? score - 2.f * slack * size_of : INFINITY;
    const float high = mine && !keep && score > -INFINITY ? score + 2.f * slack * size_of : -INFINITY;
    sure = sure && -warp_max(-low) > warp_max(high);
    unsigned kept = __ballot_sync(kAll, keep);        // bit of each kept group's first lane
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const int e = lane + 32 * i;
      if (e < p.E && !(kept >> ((e / size) << (5 - shift)) & 1u)) choice[i] = -INFINITY;
    }
  }
  // the lane's largest choice, the lowest index first
  float best = -INFINITY, best_p = 0.f;
  int best_e = 0x7fffffff;
  auto rescan = [&]() {
    best = -INFINITY; best_p = 0.f; best_e = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (choice[i] > best) { best = choice[i]; best_p = prob[i]; best_e = lane + 32 * i; }
  };
  rescan();
  float chosen = 0.f, total = 0.f, last = INFINITY, last_p = 0.f;
  int id = -1;
  for (int j = 0; j <= p.top_k; ++j) {
    const float m = warp_max(best);
    if (m == -INFINITY) break;
    if (m == INFINITY) sure = false;                   // (a bias of +inf)
    const int e = static_cast<int>(__reduce_min_sync(kAll, best == m ? static_cast<unsigned>(best_e) : 0x7fffffffu));
    const float pe = __shfl_sync(kAll, best_p, e & 31);
    // is this one surely behind the one before it?
    if (plain) {
      // different logits have different exponentials unless they are nearly equal or far out; equal ones are equal in 64 bits too
      sure = sure && (last == INFINITY || last == m || (last - m > 1e-12f && (p.sigmoid ? last < 16.f && m > -600.f : m - top > -600.f)));
      if (last == m && p.sigmoid && m <= -600.f) sure = false;
    } else {
      sure = sure && (last == INFINITY || last - m > slack * (last_p + pe + fabsf(last) + fabsf(m)));
    }
    if (j == p.top_k) break;
    last = m;
    last_p = pe;
    if (lane == j) { chosen = pe; id = e; }
    total += pe;
    if (best_e == e) {
#pragma unroll
      for (int i = 0; i < EPL; ++i)
        if (e == lane + 32 * i) choice[i] = -INFINITY;
      rescan();
    }
  }
  if (id >= 0 && total < 1e-6f) sure = false;         // weights that 32 bits may not tell from zero
  if (__ballot_sync(kAll, !sure)) {
    __syncwarp();
    route_row_64<EPL>(p, token, s_choice[warp]);
    return;
  }
  if (lane < p.top_k) {
    chosen = p.renormalize ? (total > 0.f ? chosen / total : 0.f) : chosen * inverse;
    const long long o = static_cast<long long>(token) * p.top_k + lane;
    p.weights[o] = chosen * p.scale;
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
