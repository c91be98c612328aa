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

// The definition in 64 bits, for the rows that 32 bits do not settle (one in some thousands).  One warp; lane l works on experts l,
// l + 32, ...; `scratch` has room for 2 E values: p, and the choices behind them.
__device__ __noinline__ void choices_64(const RouteParams& p, int token, double* scratch) {
  const int lane = threadIdx.x & 31;
  double* prob = scratch;
  double* choice = scratch + p.E;
  double top = kNone;
#pragma unroll 1
  for (int e = lane; e < p.E; e += 32) {
    const float l = load_logit(p.logits, p.type, static_cast<long long>(token) * p.E + e);
    const double x = l > -INFINITY ? fmin(static_cast<double>(l), 1e200) : kNone;      // +inf takes all of the softmax
    prob[e] = x;
    top = fmax(top, x);
  }
  for (int d = 16; d; d >>= 1) top = fmax(top, __shfl_xor_sync(kAll, top, d));
  double sum = 0.0;
#pragma unroll 1
  for (int e = lane; e < p.E; e += 32) {
    const double x = prob[e];
    const double v = exp(p.sigmoid ? -x : x - top);      // (of kNone: not used)
    prob[e] = x <= kNone ? -1.0 : v;
    if (x > kNone) sum += v;
  }
  for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(kAll, sum, d);
#pragma unroll 1
  for (int e = lane; e < p.E; e += 32) {
    double v = prob[e];
    const bool in = v >= 0.0;
    v = p.sigmoid ? 1.0 / (1.0 + v) : v / sum;
    prob[e] = v;
    choice[e] = !in ? kNone : p.bias ? v + static_cast<double>(__ldg(p.bias + e)) : v;
  }
  __syncwarp();
}

// The kept groups, bit n << shift for group n, from the choices.
__device__ __noinline__ unsigned groups_64(const RouteParams& p, const double* choice, int shift_out) {
  const int lane = threadIdx.x & 31, size = p.E / p.groups;
  const int shift = 5 - (32 - __clz(p.groups - 1)), per = 1 << shift;   // 2^shift lanes per group
  const int group = lane >> shift, sub = lane & (per - 1);
  double first = kNone, second = kNone;
  if (group < p.groups)
#pragma unroll 1
    for (int i = sub; i < size; i += per) {
      const double c = choice[group * size + i];
      second = fmax(second, fmin(first, c));
      first = fmax(first, c);
    }
  for (int d = 1; d < per; d <<= 1) {
    const double of = __shfl_xor_sync(kAll, first, d), os = __shfl_xor_sync(kAll, second, d);
    second = fmax(fmin(first, of), fmax(second, os));
    first = fmax(first, of);
  }
  const double score = p.group_max || second <= kNone ? first : first + second;
  int better = 0;
  for (int j = 0; j < p.groups; ++j) {
    const double other = __shfl_sync(kAll, score, j << shift);
    better += other > score || (other == score && j < group);
  }
  const unsigned kept = __ballot_sync(kAll, group < p.groups && sub == 0 && better < p.top_groups);
  if (shift == shift_out) return kept;
  unsigned moved = 0;
  for (int j = 0; j < p.groups; ++j) moved |= (kept >> (j << shift) & 1u) << (j << shift_out);
  return moved;
}

__device__ __noinline__ void route_row_64(const RouteParams& p, int token, double* scratch) {
  const int lane = threadIdx.x & 31;
  double* prob = scratch;
  double* choice = scratch + p.E;
  choices_64(p, token, scratch);
  if (p.groups > 1) {
    const int size = p.E / p.groups;
    const unsigned kept = groups_64(p, choice, 0);
    for (int e = lane; e < p.E; e += 32)
      if (!(kept >> (e / size) & 1u)) choice[e] = kNone;
    __syncwarp();
  }
  double chosen = 0.0, total = 0.0;   // lane j keeps slot j's weight
  int id = -1;
#pragma unroll 1
  for (int j = 0; j < p.top_k; ++j) {
    double best = kNone;              // the lane's largest choice, the lowest index first
    int at = 0x7fffffff;
#pragma unroll 1
    for (int e = lane; e < p.E; e += 32)
      if (choice[e] > best) { best = choice[e]; at = e; }
    // the bits of a double, made to sort like an unsigned number: the upper halves' maximum, then the lower ones' among those
    const long long bits = __double_as_longlong(best);
    const unsigned long long key = static_cast<unsigned long long>(bits ^ ((bits >> 63) | (1LL << 63)));
    const unsigned high = static_cast<unsigned>(key >> 32), low = static_cast<unsigned>(key);
    const bool in = high == __reduce_max_sync(kAll, high);
    const unsigned most = __reduce_max_sync(kAll, in ? low : 0u);
    const int e = static_cast<int>(__reduce_min_sync(kAll, in && low == most ? static_cast<unsigned>(at) : 0x7fffffffu));
    if (e == 0x7fffffff) break;       // only lanes that have nothing left
    const double pe = prob[e];
    if (lane == j) { chosen = pe; id = e; }
    total += pe;
    if (lane == (e & 31)) choice[e] = kNone;
    __syncwarp();
  }
  if (lane < p.top_k) {
    if (p.renormalize) chosen = total > 0.0 ? chosen / total : 0.0;
    const long long o = static_cast<long long>(token) * p.top_k + lane;
    p.weights[o] = static_cast<float>(chosen * static_cast<double>(p.scale));
    p.ids[o] = id;
  }
}

// One warp per token.  Where 32 bits do not settle an order, it is not taken from them:
//   * without a bias the order of the choices is that of the logits, which are compared exactly -- where different logits have
//     different p in 64 bits, else (a sigmoid of 16 and more, logits that nothing tells apart) the row is done again there;
//   * sigmoid and bias: the few candidates' choices are computed in 64 bits, one lane each;
//   * softmax and bias: each chosen one must be further from every other candidate than the two can be wrong, each by its own p
//     and choice (a large p that a negative bias takes back is wrong by far more than its choice shows), else the row is done
//     again in 64 bits;
//   * the choice of groups: the same with the groups' scores.
// Candidates: at least top_k + 1 choices are as large as the (top_k + 1)-th largest of the 32 lanes' maxima, and few more are
// (about ten in all for 8 of 256).  They go to a list in shared memory and are ranked by comparing each with all of them.
// The kernel is bound by issue, not by its bytes (72 % of the issue slots busy, one warp's dependent instructions wait for one another):
// 8 of 256 for 16384 tokens takes 14.3 us by softmax and 15.3 by sigmoid (730 instructions of a warp per token), by sigmoid with
// a bias 18.0, with eight groups and a bias 23.2 (1200 instructions), where the bytes alone take 2.7.
// FULL: there are exactly 32 * EPL experts
template <int EPL, int TYPE, bool FULL>
__global__ void __launch_bounds__(kRouteWarps * 32)
route_kernel(const RouteParams p) {
  __shared__ double s_all[kRouteWarps][EPL * 64 + 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int token = blockIdx.x * kRouteWarps + warp;
  if (token >= p.T) return;
  grid_release();
  grid_wait();
  double* scratch = s_all[warp];
  const bool fine = p.bias && p.sigmoid;   // candidates in 64 bits
  float logit[EPL], choice[EPL], prob[EPL];  // prob: exp(logit - top), or p itself where it is needed
  float top = -INFINITY;
  const long long row = static_cast<long long>(token) * p.E + lane;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    float l = -INFINITY;
    if (FULL || lane + 32 * i < p.E) l = fmaxf(load_logit(p.logits, TYPE, row + 32 * i), -INFINITY);   // NaN: -inf
    logit[i] = choice[i] = l;
    top = fmaxf(top, l);
  }
  top = warp_max(top);
  if (top == -INFINITY) {         // nothing to choose from: a row behind the last sequence, say
    if (lane < p.top_k) {
      const long long o = static_cast<long long>(token) * p.top_k + lane;
      p.weights[o] = 0.f;
      p.ids[o] = -1;
    }
    return;
  }
  bool sure = top < INFINITY;
  float inverse = 1.f;            // of the softmax's sum
  if (p.sigmoid) {
#pragma unroll
    for (int i = 0; i < EPL; ++i) prob[i] = __frcp_rn(1.f + expf(-logit[i]));
  } else {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      prob[i] = expf(logit[i] - (top > -INFINITY ? top : 0.f));     // of -inf: 0
      sum += prob[i];
    }
    sum = warp_sum(sum);
    inverse = sum > 0.f ? 1.f / sum : 0.f;
    if (p.bias || p.groups > 1) {
#pragma unroll
      for (int i = 0; i < EPL; ++i) prob[i] *= inverse;
      inverse = 1.f;
    }
  }
  if (p.bias) {
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const float v = prob[i] + (FULL || lane + 32 * i < p.E ? __ldg(p.bias + lane + 32 * i) : 0.f);
      choice[i] = logit[i] > -INFINITY ? fmaxf(v, -INFINITY) : -INFINITY;
    }
  }
  // How far 32 bits can be off, in steps of 2^-24.
  // Sigmoid: the exponential 4 of itself, which moves p by p (1 - p) <= 1/4 as much, its sum with one and the reciprocal 1 of p each:
  // 3, or 1.8e-7, in all.
  // Softmax, with d = top - logit: d of p for the rounding of d, 4 for the exponential, 26 for the sum (15 + 5 roundings and the
  // exponentials in it), its inverse 1, the product 1: (d + 32) p, taken as (d + 40) p; d is at most -ln p, and not above 104
  // where p is not zero.  It falls as p does; all of a row's p together are off by less than 41.  Below the normal numbers p is off
  // by steps of 2^-149.
  // The bias's addition: 1 of the choice.
  // (Kept close: a row that has to be done again costs ten microseconds of latency, most of it the fetching of instructions.)
  constexpr float kStep = 1.f / (1 << 24), kSigmoidOff = 1.8e-7f;
  if (p.groups > 1) {
    const int size = p.E / p.groups;
    // the two largest of each group: of group n in lane n << shift
    float first = -INFINITY, second = -INFINITY;
    int shift = 0;
    if (size == 32) {   // group i is what the lanes hold in register i
#pragma unroll
      for (int i = 0; i < EPL; ++i) {
        const float c = p.bias ? choice[i] : logit[i] > -INFINITY ? prob[i] : -INFINITY;
        const float a = warp_max(c);
        const int at = __ffs(__ballot_sync(kAll, c == a)) - 1;
        const float b = warp_max(lane == at ? -INFINITY : c);
        if (lane == i) { first = a; second = b; }
      }
    } else {
      float* s = reinterpret_cast<float*>(scratch);
#pragma unroll
      for (int i = 0; i < EPL; ++i)
        if (FULL || lane + 32 * i < p.E) s[lane + 32 * i] = p.bias ? choice[i] : logit[i] > -INFINITY ? prob[i] : -INFINITY;
      __syncwarp();
      // 2^shift lanes per group; each group starts at another place, so that the reads spread over the banks
      shift = 5 - (32 - __clz(p.groups - 1));
      const int per = 1 << shift, group = lane >> shift, sub = lane & (per - 1);
      if (group < p.groups) {
        const int n = (size - sub + per - 1) >> shift;
        int at = n > group ? group : 0;
        const float* mine = s + group * size + sub;
        for (int i = 0; i < n; ++i) {
          const float c = mine[per * at];
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
      __syncwarp();
    }
    const bool mine = (lane >> shift) < p.groups && (lane & ((1 << shift) - 1)) == 0;
    const float score = p.group_max || second == -INFINITY ? first : first + second;
    // the best top_groups of them, one after the other, equal ones in order
    float left = mine ? score : -INFINITY;
    unsigned kept = 0;                                      // bit of each kept group's first lane
    for (int j = 0; j < p.top_groups; ++j) {
      const float m = warp_max(left);
      if (m == -INFINITY) break;
      const int at = __ffs(__ballot_sync(kAll, left == m)) - 1;
      kept |= 1u << at;
      if (lane == at) left = -INFINITY;
    }
    // Every kept group must be surely better than every other.  How far a score can be off: its two p, the two choices' own
    // roundings -- of the choices, which may be large and cancel in their sum -- and the sum's.  (A choice and its error grow
    // together, so an expert that 32 bits do not put among a group's first two cannot raise the score by more.)  Twice that, for
    // the rounding of the limits themselves.
    const float next = p.group_max || second == -INFINITY ? 0.f : second;
    float off = p.sigmoid ? 2.f * kSigmoidOff : 41.f * kStep;
    if (!p.sigmoid && !p.bias)
      off = (first * (40.f + fminf(-__logf(first), 104.f)) + next * (40.f + fminf(-__logf(next), 104.f))) * kStep + 1e-37f;
    const float wrong = 2.f * (off + (fabsf(first) + fabsf(next) + fabsf(score)) * kStep);
    const float lower = wrong < INFINITY ? score - wrong : -INFINITY, upper = left > -INFINITY ? left + wrong : -INFINITY;
    const float best = warp_max(upper), worst = -warp_max(kept >> lane & 1u ? -lower : -INFINITY);
    if (!(best == -INFINITY || worst > best)) {                  // (the whole warp)
      choices_64(p, token, scratch);
      kept = groups_64(p, scratch + p.E, shift);
      __syncwarp();
    }
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const unsigned e = static_cast<unsigned>(lane + 32 * i), of = p.size_magic ? __umulhi(e, p.size_magic) : e;
      if (!(kept >> (of << shift) & 1u)) choice[i] = -INFINITY;
    }
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
  // whoever 64 bits may put above it comes along
  bound -= p.bias ? 4.f * ((fine ? kSigmoidOff : 40.f * kStep) + fabsf(bound) * kStep) : 1e-12f;
  // the list: choice and expert, logit or p, and how far the choice can be off, of each candidate; behind it the first top_k in
  // order
  float2* list = reinterpret_cast<float2*>(scratch);
  float* list_p = reinterpret_cast<float*>(scratch + EPL * 32);
  float* list_off = list_p + EPL * 32;
  float* sorted_p = list_off + EPL * 32;
  int* sorted_e = reinterpret_cast<int*>(sorted_p + 32);
  int count = 0;
  const unsigned below = (1u << lane) - 1u;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const bool in = choice[i] >= bound && choice[i] > -INFINITY;
    const unsigned votes = __ballot_sync(kAll, in);
    if (in) {
      const int at = count + __popc(votes & below);
      list[at] = make_float2(choice[i], __int_as_float(lane + 32 * i));
      list_p[at] = fine ? logit[i] : prob[i];
      if (p.bias && !fine) list_off[at] = 1.01f * kStep * ((top - logit[i] + 40.f) * prob[i] + fabsf(choice[i])) + 1e-37f;
    }
    count += __popc(votes);
  }
  __syncwarp();
  const int wanted = min(p.top_k, count);
  if (fine && count <= 32) {
    // one candidate per lane, its choice in the list's place
    double* exact = scratch;
    int e = 0;
    double pe = 0.0, mine = kNone;
    if (lane < count) {
      e = __float_as_int(list[lane].y);
      pe = 1.0 / (1.0 + exp(-static_cast<double>(list_p[lane])));
      mine = pe + static_cast<double>(__ldg(p.bias + e));
    }
    __syncwarp();
    exact[lane] = mine;
    reinterpret_cast<int*>(list_p)[lane] = e;
    __syncwarp();
    int rank = 0;
    for (int o = 0; o < count; ++o) {
      const double other = exact[o];
      rank += other > mine || (other == mine && reinterpret_cast<const int*>(list_p)[o] < e);
    }
    if (lane < count && rank < p.top_k) { sorted_p[rank] = static_cast<float>(pe); sorted_e[rank] = e; }
    sure = sure && (bound == -INFINITY || (bound > -1e30f && bound < 1e30f));   // all are here, or no bias so large that the margin
                                                                                // means nothing
  } else {
    // Without a bias.  Logits that differ have different p in 64 bits if they are more than 1e-12 apart, the larger one's p is a normal
    // number there and, of a sigmoid's, the smaller one is below 16.  `plain`: whatever differs from this one does so by more
    // (fp32 steps of 3.6e-12 at least), and it is not far out.  What is not in the list is 1e-12 below the lanes' maxima.
    const float none = p.sigmoid ? 0.f : top, most = p.sigmoid ? 16.f : INFINITY;
    bool plain = true;
    auto rank_all = [&](auto with_bias) {
      for (int c = lane; c < count; c += 32) {
        const float2 mine = list[c];
        const int e = __float_as_int(mine.y);
        const float off = decltype(with_bias)::value ? list_off[c] : 0.f;
        int rank = 0, close = 0;   // close: those that 64 bits may put on its other side, itself among them
        for (int o = 0; o < count; ++o) {
          const float2 other = list[o];
          rank += other.x > mine.x || (other.x == mine.x && __float_as_int(other.y) < e);
          if constexpr (decltype(with_bias)::value) close += !(fabsf(mine.x - other.x) > off + list_off[o]);
        }
        if (rank < p.top_k) {
          sorted_p[rank] = list_p[c];
          sorted_e[rank] = e;
          if (close > 1) sure = false;
        }
        if constexpr (!decltype(with_bias)::value) plain = plain && fabsf(mine.x) > 6.2e-5f && mine.x - none > -600.f && mine.x < most;
      }
    };
    if (p.bias) {
      rank_all(std::true_type{});
    } else {
      rank_all(std::false_type{});
      if (__any_sync(kAll, !plain)) {
        float last = INFINITY;       // place top_k; equal logits have equal p, so their ranks are the definition's
        for (int c = lane; c < count; c += 32) {
          const float mine = list[c].x;
          int before = 0;
          for (int o = 0; o < count; ++o) before += list[o].x > mine;
          if (before < p.top_k) last = fminf(last, mine);
        }
        last = -warp_max(-last);
        for (int c = lane; c < count; c += 32) {
          const float a = list[c].x;
          for (int o = 0; o < count; ++o) {
            const float b = list[o].x;
            if (a >= last && b < a) sure = sure && a - b > 1e-12f && a - none > -600.f && b < most;
          }
        }
        sure = sure && (bound == -INFINITY || (last - none > -600.f && bound < most));
      }
    }
    if (fine || (p.bias && !(bound == -INFINITY || (bound > -1e30f && bound < 1e30f)))) sure = false;
  }
  __syncwarp();
  const float chosen = lane < wanted ? sorted_p[lane] : 0.f;
  const int id = lane < wanted ? sorted_e[lane] : -1;
  const float total = warp_sum(chosen);
  if (wanted > 0 && total < 1e-6f) sure = false;      // weights that 32 bits may not tell from zero
  if (__ballot_sync(kAll, !sure)) {
    __syncwarp();
    route_row_64(p, token, scratch);
    return;
  }
  if (lane < p.top_k) {
    const float weight = p.renormalize ? (total > 0.f ? chosen / total : 0.f) : chosen * inverse;
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

// Bound by reading the rows in fp32 (4096 tokens x 8 x 2048: 268 MB, 45 us).
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
