// Quantising to the 4-bit format of int4.cuh and reading its weights back.  By the count both are bound by memory: 2 bytes of dense
// weight and half a byte of code per value, scales beside them.  Quantising 11008 x 4096 fp16 and reading it back takes 55.8 us for
// 226 MB there and back, 4.1 TB/s where a copy reaches 6.5: the quantiser's warps wait for their loads and then for issue slots
// (58 % busy with 24 warps per SM), the dequantisation's for loads (45 % busy).
//
//   symmetric     scale = round_T(max |w| / 7)                     code = clamp(rint(w / scale) + 8, 0, 15)
//   zero points   lo = min(w, 0), hi = max(w, 0)                   zero = clamp(rint(-lo / scale), 0, 15)
//                 scale = round_T((hi - lo) / 15)                  code = clamp(rint(w / scale) + zero, 0, 15)
//
// over each group, every operation rounded to fp32, rint to the nearest even number; where the scale rounds to zero the
// codes stand for zero.  A quotient of two 11-bit numbers that is not halfway between two whole numbers is further from
// there than fp32 rounds, so the codes are those of exact arithmetic.
#include <type_traits>

#include "int4.cuh"

namespace vqg {
namespace {

constexpr int kThreads = 256;

template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
  if constexpr (BF16) return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
  else return __half22float2(*reinterpret_cast<const __half2*>(&v));
}

// 32 bytes with one access where the address allows it (`wide`: it is a multiple of 32)
__device__ __forceinline__ void load32(const void* p, bool wide, uint32_t (&v)[8]) {
  if (wide) {
    asm volatile("ld.global.nc.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]) : "l"(p));
  } else {
    const uint4 a = __ldg(static_cast<const uint4*>(p)), b = __ldg(static_cast<const uint4*>(p) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
}
__device__ __forceinline__ void store32(void* p, bool wide, const uint32_t (&v)[8]) {
  if (wide) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                 ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
  } else {
    static_cast<uint4*>(p)[0] = make_uint4(v[0], v[1], v[2], v[3]);
    static_cast<uint4*>(p)[1] = make_uint4(v[4], v[5], v[6], v[7]);
  }
}

// From 192 + w / s (a multiple of 2^-16): w / s rounded to the nearest whole number, halves to the even one, plus the zero point,
// held to 0 ... 15; in the low byte.  12582912 = 1.5 * 2^23 is even, and sums around it have no bits below one.
__device__ __forceinline__ uint32_t code_of(float q192, float zero) {
  const float r = (q192 + (12582912.f - 192.f)) + zero;
  return __float_as_uint(fminf(fmaxf(r, 12582912.f), 12582927.f));
}

__device__ __noinline__ float quotient(float a, float b) { return __fdiv_rn(a, b); }

template <bool BF16>
__global__ void __launch_bounds__(kThreads)
int4_dequant_kernel(const Int4Weight w, void* __restrict__ out, bool wide) {
  using I = Int4Type<BF16>;
  const int lane = threadIdx.x & 31, g = lane & 7, t = lane >> 3;
  const long long tiles = static_cast<long long>(w.row_tiles()) * w.k_tiles();
  grid_release();
  grid_wait();
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
      store32(dst + static_cast<long long>(row) * w.K + k, wide, v);
    }
  }
}

// One unit of work is 16 rows x SPAN tile columns of 64: whole groups of 32, 64 or SPAN * 64 columns.  Lane t*8 + g reads columns
// 16t ... +15 of rows g and g + 8 of each tile, the values whose codes its 16 bytes hold, and keeps them in registers between
// the extremes and the codes, so the weight is read once.  (SPAN = 0: groups of more columns than registers hold; a second read
// that the caches serve.)
//
// The division: w / s is w * (1 / s) but for a few steps of 2^-23, and a quotient of two 11-bit numbers is either halfway between
// two whole numbers or at least 2^-13 from there; rounding the product to multiples of 2^-16 first (adding 192 does) turns
// what is nearly halfway into exactly halfway, and the codes are those of the correctly rounded division.
template <bool BF16, bool ZEROS, int SPAN>
__global__ void __launch_bounds__(kThreads, SPAN == 2 ? 3 : 4)
int4_quantize_kernel(const void* __restrict__ src, uint8_t* __restrict__ packed, void* __restrict__ scales,
                     uint8_t* __restrict__ zeros, int N, int K, int group, int span_all, bool wide) {
  using I = Int4Type<BF16>;
  using T = typename I::T;
  constexpr int HOLD = SPAN > 0 ? SPAN : 1;
  const int lane = threadIdx.x & 31, g = lane & 7, t = lane >> 3;
  const int span = SPAN > 0 ? SPAN : span_all;
  const int row_tiles = (N + 15) / 16, k_tiles = (K + 63) / 64, spans = (k_tiles + span - 1) / span;
  const long long unit = static_cast<long long>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  if (unit >= static_cast<long long>(row_tiles) * spans) return;
  grid_release();
  grid_wait();
  const int tr = static_cast<int>(unit / spans), kt0 = static_cast<int>(unit % spans) * span;
  const int kt1 = min(kt0 + span, k_tiles);
  const int e = blockIdx.y;
  const T* w = static_cast<const T*>(src) + static_cast<long long>(e) * N * K;
  uint8_t* codes = packed + static_cast<long long>(e) * row_tiles * k_tiles * 512;
  const long long sbase = static_cast<long long>(e) * (K / group) * N;
  const T* at[2] = {w + static_cast<long long>(min(tr * 16 + g, N - 1)) * K + t * 16, w + static_cast<long long>(min(tr * 16 + 8 + g, N - 1)) * K + t * 16};

  uint32_t v[HOLD][2][8];
  auto load = [&](int kt, uint32_t (&d)[2][8]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (kt < k_tiles && kt * 64 + t * 16 < K) {
        load32(at[h] + kt * 64, wide, d[h]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) d[h][i] = 0;
      }
    }
  };
  float lo[2] = {0.f, 0.f}, hi[2] = {0.f, 0.f};
  auto extremes = [&](const uint32_t (&d)[2][8]) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 f = unpack2<BF16>(d[h][i]);
        if (ZEROS) { lo[h] = fminf(lo[h], fminf(f.x, f.y)); hi[h] = fmaxf(hi[h], fmaxf(f.x, f.y)); }
        else hi[h] = fmaxf(hi[h], fmaxf(fabsf(f.x), fabsf(f.y)));
      }
  };
  if constexpr (SPAN > 0) {
#pragma unroll
    for (int k = 0; k < SPAN; ++k) load(kt0 + k, v[k]);
#pragma unroll
    for (int k = 0; k < SPAN; ++k) extremes(v[k]);
  } else {
    for (int kt = kt0; kt < kt1; ++kt) { load(kt, v[0]); extremes(v[0]); }
  }
  float inv[2], dv[2], z[2];
  bool tiny = false;
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
    const float s = I::to_float(st);
    const float d = s > 0.f ? s : 1.f;
    z[h] = ZEROS ? fminf(fmaxf(rintf(__fdiv_rn(-lo[h], d)), 0.f), 15.f) : 8.f;
    inv[h] = __fdiv_rn(1.f, d);
    dv[h] = d;
    tiny = tiny || inv[h] > 1e38f;
    const int row = tr * 16 + h * 8 + g, k = kt0 * 64 + t * 16;
    if (row < N && k < K && (group == 32 ? (t & 1) == 0 : t == 0)) {
      const long long to = sbase + static_cast<long long>(k / group) * N + row;
      static_cast<T*>(scales)[to] = st;
      if (ZEROS) zeros[to] = static_cast<uint8_t>(z[h]);
    }
  }
  tiny = __any_sync(0xffffffffu, tiny);
  auto encode = [&](int kt, const uint32_t (&d)[2][8]) {
    uint32_t words[4] = {0, 0, 0, 0};
    if (!tiny) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 8; ++i) {   // pair i: word i / 2, q = i % 2
          const float2 f = unpack2<BF16>(d[h][i]);
          const uint32_t pair = __byte_perm(code_of(__fmaf_rn(f.x, inv[h], 192.f), z[h]), code_of(__fmaf_rn(f.y, inv[h], 192.f), z[h]), 0x1410);
          words[i >> 1] |= pair << (8 * (i & 1) + 4 * h);
        }
    } else {                            // 1 / s is not a number that 32 bits hold
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int h = i >> 3, j = i & 7;
        const float2 f = unpack2<BF16>(d[h][j]);
        const uint32_t pair = __byte_perm(code_of(quotient(f.x, dv[h]) + 192.f, z[h]), code_of(quotient(f.y, dv[h]) + 192.f, z[h]), 0x1410);
        words[j >> 1] |= pair << (8 * (j & 1) + 4 * h);
      }
    }
    reinterpret_cast<uint4*>(codes + (static_cast<long long>(tr) * k_tiles + kt) * 512)[lane] =
        make_uint4(words[0], words[1], words[2], words[3]);
  };
  if constexpr (SPAN > 0) {
#pragma unroll
    for (int k = 0; k < SPAN; ++k)
      if (kt0 + k < k_tiles) encode(kt0 + k, v[k]);
  } else {
    for (int kt = kt0; kt < kt1; ++kt) { load(kt, v[0]); encode(kt, v[0]); }
  }
}

}  // namespace

int launch_int4_dequant(const Int4Weight& w, void* out, int experts, bool bf16, cudaStream_t s) {
  const long long tiles = static_cast<long long>(w.row_tiles()) * w.k_tiles();
  const long long want = (tiles + kThreads / 32 - 1) / (kThreads / 32), most = 8LL * sm_count_cached();
  const dim3 grid(static_cast<unsigned>(want < most ? want : most), experts);
  const bool wide = reinterpret_cast<uintptr_t>(out) % 32 == 0;   // rows are multiples of 64 bytes
  return cuda_status(bf16 ? launch_ahead(int4_dequant_kernel<true>, grid, kThreads, 0, s, false, w, out, wide)
                          : launch_ahead(int4_dequant_kernel<false>, grid, kThreads, 0, s, false, w, out, wide));
}

int launch_int4_quantize(const void* w, uint8_t* packed, void* scales, uint8_t* zeros, int experts, int N, int K, int group,
                         bool bf16, cudaStream_t s) {
  const int k_tiles = (K + 63) / 64, span = group >= K ? k_tiles : group == 32 ? 1 : group / 64;
  const long long units = static_cast<long long>((N + 15) / 16) * ((k_tiles + span - 1) / span);
  const long long blocks = (units + kThreads / 32 - 1) / (kThreads / 32);
  if (blocks > 0x7fffffffLL) return VQG_ERR_UNSUPPORTED;
  const dim3 grid(static_cast<unsigned>(blocks), experts);
  const bool wide = reinterpret_cast<uintptr_t>(w) % 32 == 0;
  auto go = [&](auto kernel) {
    return cuda_status(launch_ahead(kernel, grid, kThreads, 0, s, false, w, packed, scales, zeros, N, K, group, span, wide));
  };
  auto with = [&](auto n) {
    constexpr int S = decltype(n)::value;
    if (zeros) return bf16 ? go(int4_quantize_kernel<true, true, S>) : go(int4_quantize_kernel<false, true, S>);
    return bf16 ? go(int4_quantize_kernel<true, false, S>) : go(int4_quantize_kernel<false, false, S>);
  };
  if (span == 1) return with(std::integral_constant<int, 1>{});
  if (span == 2) return with(std::integral_constant<int, 2>{});
  return with(std::integral_constant<int, 0>{});
}

}  // namespace vqg
