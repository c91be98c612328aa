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
#include <type_traits>

#include "int4.cuh"

namespace vqg {
namespace {

constexpr int kRouteWarps = 4;
constexpr unsigned kAll = 0xffffffffu;
constexpr double kNone = -1e300;   // choice of an expert that cannot be chosen, in 64 bits; -inf in 32

// type: 0 fp16, 1 bf16, 2 fp32
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
  unsigned size_magic;   // e / (E / groups) = e * size_magic >> 32 for e < 512: ceil(2^32 / size); 0 for a size of one
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
// exactly.
//
// Selection: at least top_k + 1 choices are as large as the (top_k + 1)-th largest of the 32 lanes' maxima, and few more are
// (about ten in all for 8 of 256).  Those go to a list in shared memory and are ranked by comparing each with all of them.
// The kernel is bound by issue, not by its bytes.
// FULL: there are exactly 32 * EPL experts
template <int EPL, int TYPE, bool FULL>
__global__ void __launch_bounds__(kRouteWarps * 32)
route_kernel(const RouteParams p) {
  __shared__ double s_all[kRouteWarps][EPL * 32 + EPL * 16 + 50];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int token = blockIdx.x * kRouteWarps + warp;
  if (token >= p.T) return;
  grid_release();
  grid_wait();
  double* scratch = s_all[warp];
  const bool plain = !p.bias && p.groups == 1;
  float choice[EPL], prob[EPL];   // prob: exp(logit - top) or the sigmoid
  float top = -INFINITY;
  const long long row = static_cast<long long>(token) * p.E + lane;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    float l = -INFINITY;
    if (FULL || lane + 32 * i < p.E) l = fmaxf(load_logit(p.logits, TYPE, row + 32 * i), -INFINITY);   // NaN: -inf
    choice[i] = l;
    top = fmaxf(top, l);
  }
  top = warp_max(top);
  bool sure = top < INFINITY;
  float inverse = 1.f;            // of the softmax's sum
  if (p.sigmoid) {
#pragma unroll
    for (int i = 0; i < EPL; ++i) prob[i] = __fdividef(1.f, 1.f + expf(-choice[i]));
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
  // 32-bit errors, relative to p: the exponential 2^-22, its sum with one 2^-24, the reciprocal 2^-22; in the softmax also the
  // exponent's difference (at most 2^-25 of it, times what is left of p) and a sum of at most 16 + 5 roundings.  Adding the bias
  // rounds once more.  `slack` is twice what that comes to, relative to what goes in.
  const float slack = p.sigmoid ? 1.f / (1 << 20) : 1.f / (1 << 18);
  if (!plain) {
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      if (choice[i] > -INFINITY) {
        prob[i] *= inverse;
        choice[i] = p.bias ? fmaxf(prob[i] + __ldg(p.bias + lane + 32 * i), -INFINITY) : prob[i];
      }
    }
    inverse = 1.f;
  }
  if (p.groups > 1) {
    const int size = p.E / p.groups;
    float* s = reinterpret_cast<float*>(scratch);
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (FULL || lane + 32 * i < p.E) s[lane + 32 * i] = choice[i];
    __syncwarp();
    // 32 / 2^n lanes per group, 2^n >= groups; each starts at another place, so that the groups' reads spread over the banks
    const int shift = 32 - __clz(p.groups - 1), per = 32 >> shift;   // lanes per group
    const int group = lane >> (5 - shift), sub = lane & (per - 1);
    float first = -INFINITY, second = -INFINITY;
    if (group < p.groups) {
      const int n = (size - sub + per - 1) >> (5 - shift);
      int at = n > group ? group : 0;
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
    const unsigned kept = __ballot_sync(kAll, keep);        // bit of each kept group's first lane
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const unsigned e = static_cast<unsigned>(lane + 32 * i), of = p.size_magic ? __umulhi(e, p.size_magic) : e;
      if (!(kept >> (of << (5 - shift)) & 1u)) choice[i] = -INFINITY;
    }
    __syncwarp();
  }
  // the (top_k + 1)-th largest of the lanes' maxima
  float bound = -INFINITY;
  if (p.top_k < 32) {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < EPL; ++i) m = fmaxf(m, choice[i]);
    // (lanes whose maxima are equal leave together: the bound is then lower, never higher)
    for (int j = 0; j <= p.top_k; ++j) {
      bound = warp_max(m);
      if (m == bound) m = -INFINITY;
    }
  }
  // the list: choice and expert, and p, of each candidate; behind it the first top_k + 1 in order
  float2* list = reinterpret_cast<float2*>(scratch);
  float* list_p = reinterpret_cast<float*>(scratch + EPL * 32);
  float* sorted_c = list_p + EPL * 32;
  float* sorted_p = sorted_c + 33;
  int* sorted_e = reinterpret_cast<int*>(sorted_p + 33);
  int count = 0;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const bool in = choice[i] >= bound && choice[i] > -INFINITY;
    const unsigned votes = __ballot_sync(kAll, in);
    if (in) {
      const int at = count + __popc(votes & ((1u << lane) - 1u));
      list[at] = make_float2(choice[i], __int_as_float(lane + 32 * i));
      list_p[at] = prob[i];
    }
    count += __popc(votes);
  }
  __syncwarp();
  const int wanted = min(p.top_k, count);
  for (int c = lane; c < count; c += 32) {
    const float2 mine = list[c];
    const int e = __float_as_int(mine.y);
    int rank = 0;
    for (int o = 0; o < count; ++o) {
      const float2 other = list[o];
      rank += other.x > mine.x || (other.x == mine.x && __float_as_int(other.y) < e);
    }
    if (rank <= p.top_k) { sorted_c[rank] = mine.x; sorted_p[rank] = list_p[c]; sorted_e[rank] = e; }
  }
  __syncwarp();
  const float chosen_p = lane < wanted ? sorted_p[lane] : 0.f;
  const int id = lane < wanted ? sorted_e[lane] : -1;
  if (lane + 1 < min(count, p.top_k + 1)) {   // is number lane + 1 surely behind number lane?
    const float a = sorted_c[lane], b = sorted_c[lane + 1];
    if (plain)   // different logits have different exponentials unless they are nearly equal or far out; equal ones are equal in 64 bits too
      sure = sure && (p.sigmoid ? b > -600.f && (a == b || (a - b > 1e-12f && a < 16.f)) : a == b || (a - b > 1e-12f && b - top > -600.f));
    else
      sure = sure && a < INFINITY && a - b > slack * (sorted_p[lane] + sorted_p[lane + 1] + fabsf(a) + fabsf(b));
  }
  const float total = warp_sum(chosen_p);
  if (wanted > 0 && total < 1e-6f) sure = false;      // weights that 32 bits may not tell from zero
  if (__ballot_sync(kAll, !sure)) {
    __syncwarp();
    route_row_64<EPL>(p, token, scratch);
    return;
  }
  if (lane < p.top_k) {
    const float weight = p.renormalize ? (total > 0.f ? chosen_p / total : 0.f) : chosen_p * inverse;
    const long long o = static_cast<long long>(token) * p.top_k + lane;
    p.weights[o] = weight * p.scale;
    p.ids[o] = id;
  }
}

// Slots by expert, one cluster of blocks: every block counts its share of the slots in shared memory, reads the others' counts from
// theirs, and so knows where its rows of each expert begin; places within that by atomics.  The order of an expert's rows
// depends on the atomics; no result does, every row of a product being computed on its own.
constexpr int kPlanThreads = 1024, kPlanBlocks = 8;
__device__ __forceinline__ int cluster_load(const int* local, int rank) {
  uint32_t at;
  int v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(local)), "r"(rank));
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__global__ void __launch_bounds__(kPlanThreads)
expert_plan_kernel(const int* __restrict__ ids, int slots, int E, int chunk_rows, int* __restrict__ row_slot,
                   int4* __restrict__ chunks, int* __restrict__ n_chunks) {
  __shared__ int count[512], place[512], scan[2][16];
  const int blocks = gridDim.x, me = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  grid_release();
  grid_wait();
  if (tid < 512) count[tid] = 0;
  __syncthreads();
  const int begin = static_cast<int>(static_cast<long long>(slots) * me / blocks), end = static_cast<int>(static_cast<long long>(slots) * (me + 1) / blocks);
  for (int i = begin + tid; i < end; i += kPlanThreads) {
    const int e = ids[i];
    if (e >= 0 && e < E) atomicAdd(count + e, 1);
  }
  if (blocks > 1) cluster_sync(); else __syncthreads();
  // thread e: rows of expert e in all, and in the blocks before this one; then rows and chunks of the experts before it
  int all = 0, before = 0, rows = 0, parts = 0;
  if (tid < 512) {
    if (tid < E) {
      for (int b = 0; b < blocks; ++b) {
        const int c = b == me ? count[tid] : cluster_load(count + tid, b);
        if (b < me) before += c;
        all += c;
      }
    }
    rows = all;
    parts = (all + chunk_rows - 1) / chunk_rows;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int r = __shfl_up_sync(kAll, rows, d), c = __shfl_up_sync(kAll, parts, d);
      if (lane >= d) { rows += r; parts += c; }
    }
    if (lane == 31) { scan[0][warp] = rows; scan[1][warp] = parts; }
  }
  __syncthreads();
  if (tid < 512) {
    for (int k = 0; k < warp; ++k) { rows += scan[0][k]; parts += scan[1][k]; }
    if (me == 0 && tid == 511) { n_chunks[0] = parts; n_chunks[1] = rows; }
    rows -= all;
    parts -= (all + chunk_rows - 1) / chunk_rows;
    place[tid] = rows + before;
    if (me == 0)
      for (int i = 0; i < all; i += chunk_rows) chunks[parts++] = make_int4(tid, rows + i, min(chunk_rows, all - i), 0);
  }
  __syncthreads();
  for (int i = begin + tid; i < end; i += kPlanThreads) {
    const int e = ids[i];
    if (e >= 0 && e < E) row_slot[atomicAdd(place + e, 1)] = i;
  }
  if (blocks > 1) cluster_sync();   // nobody leaves while its counts may be read
}

template <bool BF16>
__global__ void __launch_bounds__(256)
expert_combine_kernel(const float* __restrict__ part, const ExpertRows rows, void* __restrict__ y, int cols) {
  using I = Int4Type<BF16>;
  const int token = blockIdx.x;
  grid_release();
  grid_wait();
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
                renormalize ? 1 : 0, scale, 0};
  const int size = E / groups;
  p.size_magic = size > 1 ? static_cast<unsigned>(((1ULL << 32) + size - 1) / size) : 0u;
  const int blocks = (T + kRouteWarps - 1) / kRouteWarps;
  auto go = [&](auto kernel) {
    return cuda_status(launch_ahead(kernel, dim3(blocks), kRouteWarps * 32, 0, s, false, p));
  };
  auto with = [&](auto type) {
    constexpr int Y = decltype(type)::value;
    if (E <= 32) return go(route_kernel<1, Y, false>);
    if (E <= 64) return E == 64 ? go(route_kernel<2, Y, true>) : go(route_kernel<2, Y, false>);
    if (E <= 128) return E == 128 ? go(route_kernel<4, Y, true>) : go(route_kernel<4, Y, false>);
    if (E <= 256) return E == 256 ? go(route_kernel<8, Y, true>) : go(route_kernel<8, Y, false>);
    return E == 512 ? go(route_kernel<16, Y, true>) : go(route_kernel<16, Y, false>);
  };
  if (E > 512) return static_cast<int>(VQG_ERR_UNSUPPORTED);
  if (logits_type == 0) return with(std::integral_constant<int, 0>{});
  if (logits_type == 1) return with(std::integral_constant<int, 1>{});
  return with(std::integral_constant<int, 2>{});
}

int launch_expert_plan(const int* ids, int slots, int E, int chunk_rows, int* row_slot, int4* chunks, int* n_chunks,
                       cudaStream_t s) {
  // one block for a few thousand slots, a cluster of eight above (one block took 25 us for 32768 slots)
  cudaLaunchConfig_t cfg{};
  const int blocks = slots > 4 * kPlanThreads ? kPlanBlocks : 1;
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(kPlanThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = blocks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, expert_plan_kernel, ids, slots, E, chunk_rows, row_slot, chunks, n_chunks);
  count_launch();
  return cuda_status(e);
}

int launch_expert_combine(const float* part, const ExpertRows& rows, void* y, int tokens, int cols, bool bf16, cudaStream_t s) {
  return cuda_status(bf16 ? launch_ahead(expert_combine_kernel<true>, dim3(tokens), 256, 0, s, false, part, rows, y, cols)
                          : launch_ahead(expert_combine_kernel<false>, dim3(tokens), 256, 0, s, false, part, rows, y, cols));
}

}  // namespace vqg
