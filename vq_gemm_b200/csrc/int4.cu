// Quantising to the 4-bit format of int4.cuh and reading its weights back.  Both are bound by memory: 2 bytes of dense
// weight and half a byte of code per value, scales beside them.
//
//   symmetric     scale = round_T(max |w| / 7)                     code = clamp(rint(w / scale) + 8, 0, 15)
//   zero points   lo = min(w, 0), hi = max(w, 0)                   zero = clamp(rint(-lo / scale), 0, 15)
//                 scale = round_T((hi - lo) / 15)                  code = clamp(rint(w / scale) + zero, 0, 15)
//
// over each group, every operation rounded to fp32, rint to the nearest even number; where the scale rounds to zero the
// codes stand for zero.  A quotient of two 11-bit numbers that is not halfway between two whole numbers is further from
// there than fp32 rounds, so the codes are those of exact arithmetic.
#include "int4.cuh"

namespace vqg {
namespace {

constexpr int kThreads = 256;

template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
  if constexpr (BF16) return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
  else return __half22float2(*reinterpret_cast<const __half2*>(&v));
}

template <bool BF16>
__global__ void __launch_bounds__(kThreads)
int4_dequant_kernel(const Int4Weight w, void* __restrict__ out) {
  using I = Int4Type<BF16>;
  const int lane = threadIdx.x & 31, g = lane & 7, t = lane >> 3;
  const long long tiles = static_cast<long long>(w.row_tiles()) * w.k_tiles();
  const int e = blockIdx.y;
  const uint8_t* packed = w.packed + e * w.expert_bytes();
  const uint8_t* zeros = w.zeros ? w.zeros + e * w.expert_scales() : nullptr;
  unsigned short* dst = static_cast<unsigned short*>(out) + static_cast<long long>(e) * w.N * w.K;
  for (long long tile = static_cast<long long>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5); tile < tiles;
       tile += static_cast<long long>(gridDim.x) * (kThreads / 32)) {
    const int tr = static_cast<int>(tile / w.k_tiles()), kt = static_cast<int>(tile % w.k_tiles());
    const int k = kt * 64 + t * 16;
    if (k >= w.K) continue;
    const uint4 c = __ldg(reinterpret_cast<const uint4*>(packed + tile * 512) + lane);
    const uint32_t words[4] = {c.x, c.y, c.z, c.w};
    const long long at = static_cast<long long>(int4_group_of(w, k)) * w.N + static_cast<long long>(e) * w.expert_scales();
    const long long atz = static_cast<long long>(int4_group_of(w, k)) * w.N;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = tr * 16 + h * 8 + g;
      if (row >= w.N) continue;
      const uint32_t s2 = int4_scale2<BF16>(w.scales, at + row);
      const uint32_t off = I::offset(zeros ? (__ldg(zeros + atz + row) & 15) : 8);
      uint32_t v[8];
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        v[2 * s] = h ? int4_pair<BF16, 1, 0>(words[s], off, s2) : int4_pair<BF16, 0, 0>(words[s], off, s2);
        v[2 * s + 1] = h ? int4_pair<BF16, 1, 1>(words[s], off, s2) : int4_pair<BF16, 0, 1>(words[s], off, s2);
      }
      uint4* d = reinterpret_cast<uint4*>(dst + static_cast<long long>(row) * w.K + k);
      d[0] = make_uint4(v[0], v[1], v[2], v[3]);
      d[1] = make_uint4(v[4], v[5], v[6], v[7]);
    }
  }
}

// A warp owns 16 rows x `span` tile columns: whole groups (span = group / 64, or 1 where the group is 32, or the whole row).
// Lane t*8 + g reads columns 16t ... +15 of rows g and g + 8 of each tile: the values whose codes its 16 bytes hold.
template <bool BF16, bool ZEROS>
__global__ void __launch_bounds__(kThreads)
int4_quantize_kernel(const void* __restrict__ src, uint8_t* __restrict__ packed, void* __restrict__ scales,
                     uint8_t* __restrict__ zeros, int N, int K, int group, int span) {
  using I = Int4Type<BF16>;
  using T = typename I::T;
  const int lane = threadIdx.x & 31, g = lane & 7, t = lane >> 3;
  const int row_tiles = (N + 15) / 16, k_tiles = (K + 63) / 64, spans = (k_tiles + span - 1) / span;
  const long long unit = static_cast<long long>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  if (unit >= static_cast<long long>(row_tiles) * spans) return;
  const int tr = static_cast<int>(unit / spans), kt0 = static_cast<int>(unit % spans) * span;
  const int kt1 = min(kt0 + span, k_tiles);
  const int e = blockIdx.y;
  const T* w = static_cast<const T*>(src) + static_cast<long long>(e) * N * K;
  uint8_t* codes = packed + static_cast<long long>(e) * row_tiles * k_tiles * 512;
  const long long sbase = static_cast<long long>(e) * (K / group) * N;

  auto load = [&](int kt, int h, uint32_t (&v)[8]) {
    const int row = tr * 16 + h * 8 + g, k = kt * 64 + t * 16;
    uint4 a = make_uint4(0, 0, 0, 0), b = a;
    if (row < N && k < K) {
      const uint4* p = reinterpret_cast<const uint4*>(w + static_cast<long long>(row) * K + k);
      a = __ldg(p); b = __ldg(p + 1);
    }
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  };
  float lo[2] = {0.f, 0.f}, hi[2] = {0.f, 0.f};
  for (int kt = kt0; kt < kt1; ++kt)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t v[8];
      load(kt, h, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 f = unpack2<BF16>(v[i]);
        if (ZEROS) { lo[h] = fminf(lo[h], fminf(f.x, f.y)); hi[h] = fmaxf(hi[h], fmaxf(f.x, f.y)); }
        else hi[h] = fmaxf(hi[h], fmaxf(fabsf(f.x), fabsf(f.y)));
      }
    }
  float s[2], z[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    // a group of 32 columns is two threads t, a longer one all four
    hi[h] = fmaxf(hi[h], __shfl_xor_sync(0xffffffffu, hi[h], 8));
    if (group != 32) hi[h] = fmaxf(hi[h], __shfl_xor_sync(0xffffffffu, hi[h], 16));
    if (ZEROS) {
      lo[h] = fminf(lo[h], __shfl_xor_sync(0xffffffffu, lo[h], 8));
      if (group != 32) lo[h] = fminf(lo[h], __shfl_xor_sync(0xffffffffu, lo[h], 16));
    }
    const T st = I::from_float(ZEROS ? __fdiv_rn(hi[h] - lo[h], 15.f) : __fdiv_rn(hi[h], 7.f));
    s[h] = I::to_float(st);
    const float d = s[h] > 0.f ? s[h] : 1.f;
    z[h] = ZEROS ? fminf(fmaxf(rintf(__fdiv_rn(-lo[h], d)), 0.f), 15.f) : 8.f;
    const int row = tr * 16 + h * 8 + g, k = kt0 * 64 + t * 16;
    if (row < N && k < K && (group == 32 ? (t & 1) == 0 : t == 0)) {
      const long long at = sbase + static_cast<long long>(k / group) * N + row;
      static_cast<T*>(scales)[at] = st;
      if (ZEROS) zeros[at] = static_cast<uint8_t>(z[h]);
    }
    s[h] = d;
  }
  for (int kt = kt0; kt < kt1; ++kt) {
    uint32_t words[4] = {0, 0, 0, 0};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t v[8];
      load(kt, h, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) {   // pair i: word i / 2, q = i % 2
        const float2 f = unpack2<BF16>(v[i]);
        const uint32_t c0 = static_cast<uint32_t>(fminf(fmaxf(rintf(__fdiv_rn(f.x, s[h])) + z[h], 0.f), 15.f));
        const uint32_t c1 = static_cast<uint32_t>(fminf(fmaxf(rintf(__fdiv_rn(f.y, s[h])) + z[h], 0.f), 15.f));
        words[i >> 1] |= (c0 | (c1 << 16)) << (8 * (i & 1) + 4 * h);
      }
    }
    reinterpret_cast<uint4*>(codes + (static_cast<long long>(tr) * k_tiles + kt) * 512)[lane] =
        make_uint4(words[0], words[1], words[2], words[3]);
  }
}

int sm_count() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms > 0 ? sms : 148;
}

}  // namespace

int launch_int4_dequant(const Int4Weight& w, void* out, int experts, bool bf16, cudaStream_t s) {
  const long long tiles = static_cast<long long>(w.row_tiles()) * w.k_tiles();
  const long long want = (tiles + kThreads / 32 - 1) / (kThreads / 32), most = 8LL * sm_count();
  const dim3 grid(static_cast<unsigned>(want < most ? want : most), experts);
  if (bf16) int4_dequant_kernel<true><<<grid, kThreads, 0, s>>>(w, out);
  else int4_dequant_kernel<false><<<grid, kThreads, 0, s>>>(w, out);
  count_launch();
  return cuda_status(cudaGetLastError());
}

int launch_int4_quantize(const void* w, uint8_t* packed, void* scales, uint8_t* zeros, int experts, int N, int K, int group,
                         bool bf16, cudaStream_t s) {
  const int k_tiles = (K + 63) / 64, span = group >= K ? k_tiles : group == 32 ? 1 : group / 64;
  const long long units = static_cast<long long>((N + 15) / 16) * ((k_tiles + span - 1) / span);
  const long long blocks = (units + kThreads / 32 - 1) / (kThreads / 32);
  if (blocks > 0x7fffffffLL) return VQG_ERR_UNSUPPORTED;
  const dim3 grid(static_cast<unsigned>(blocks), experts);
  auto go = [&](auto kernel) {
    kernel<<<grid, kThreads, 0, s>>>(w, packed, scales, zeros, N, K, group, span);
    count_launch();
    return cuda_status(cudaGetLastError());
  };
  if (zeros) return bf16 ? go(int4_quantize_kernel<true, true>) : go(int4_quantize_kernel<false, true>);
  return bf16 ? go(int4_quantize_kernel<true, false>) : go(int4_quantize_kernel<false, false>);
}

}  // namespace vqg
