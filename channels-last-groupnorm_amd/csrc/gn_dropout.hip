// Dropout from a counter-based generator, with the residual's addition behind it (declared in include/gnnhwc_tokens.h): kernel
// and C ABI.
//
//   y[e] = (bits(e) >= t ? x[e] f : 0) + r[e],   t = round(65536 p),  f = 65536 / (65536 - t), rounded to float32 (float64)
// bits(e): 16 bits of Philox 4x32 with 7 rounds (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011;
// their tests find nothing against 7), counter (e / 8, offset), key the seed; element e has half e % 2, the lower first, of word
// e / 2 % 4.  No mask is stored: the backward is the same call on the gradient, without a residual.
//
// Memory bounds it as long as the generator hides behind it: 7 rounds of two 64-bit products are about 50 cycles of a SIMD
// for each of a lane's 8 elements of 16 bits, where 32 bits an element and 10 rounds would take three times as much.  float16 (65536,
// 2560): 109 us, 6.1 TB/s (a copy of that size 5.1); bfloat16 (16384, 1280) with a residual 19 us; float32 (5883, 1001) 9.1 in a
// training pass, 5.8 where x lies in the memory-side cache.  float64 (16384, 1280): 216 us, 1.6 TB/s (a lane's 64 bytes in four accesses
// that a wavefront has 64 bytes apart).
#include <math.h>
#include <stdint.h>
#include "gn_rms.h"
#include "gn_error.h"

namespace gn {
namespace {

constexpr int kGroup = 8;  // elements of one counter
struct DropoutArgs {
  const void *x, *residual;
  void *y;
  int64_t n;
  const int64_t *seed_at;  // read when the kernel runs, instead of seed
  uint64_t seed, offset;
  uint32_t least;
  double scale;
};

__device__ __forceinline__ u32x4 random_words(uint64_t counter, uint64_t offset, uint64_t seed) {
  uint32_t c0 = (uint32_t)counter, c1 = (uint32_t)(counter >> 32), c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 7; ++r) {
    const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return u32x4{c0, c1, c2, c3};
}
__device__ __forceinline__ bool kept(const u32x4 &w, int i, uint32_t least) { return (i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu) >= least; }

// The value of the lane beside this one: 0 and 1, 2 and 3, ...
__device__ __forceinline__ uint32_t neighbours(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, true); }

// One group a lane: more of them on their way at once are slower (float16 (65536, 2560) 111 us, by four 117; float32 (5883, 1001), x in the cache, 6.3, by two
// 8.1, by four 11).
template <typename T, bool RES> __global__ __launch_bounds__(kBlock) void dropout_kernel(const DropoutArgs a) {
  using A = acc_of_t<T>;
  constexpr int VEC = vec_of<T>::value, PARTS = kGroup / VEC;
  using LV = LaneVec<T, VEC>;
  const T *x = (const T *)a.x, *res = (const T *)a.residual;
  T *y = (T *)a.y;
  const uint64_t seed = a.seed_at ? (uint64_t)load_global<int64_t>(a.seed_at) : a.seed;
  const A scale = (A)a.scale;
  const int64_t group = (int64_t)blockIdx.x * kBlock + threadIdx.x;
  if ((int64_t)(blockIdx.x + 1) * (kBlock * kGroup) <= a.n) {
    // Part v of a lane's elements, and the two halves of a word each that decide on them.  float32: a group's 32 bytes are two lanes',
    // so that a wavefront reads and writes whole lines.  Of its 64 groups two neighbours make the bits of one of the first half and
    // one of the second, and hand each other what the other's elements need.  (float32 (65536, 1280) 183 us by 32 bytes a lane,
    // 110 so)
    constexpr bool kPairs = sizeof(T) == 4;
    const int lane = threadIdx.x & 63, odd = lane & 1;
    const int64_t base = group - lane;
    auto place = [&](int v) { return kPairs ? (base + v * 32) * kGroup + lane * 4 : group * kGroup + v * VEC; };
    typename LV::raw_t rx[PARTS], rr[RES ? PARTS : 1];
#pragma unroll
    for (int v = 0; v < PARTS; ++v) {
      rx[v] = load_loose<LV>(x + place(v));
      if constexpr (RES) rr[v] = load_loose<LV>(res + place(v));
    }
    u32x4 w = random_words((uint64_t)(kPairs ? base + odd * 32 + lane / 2 : group), a.offset, seed);
    if constexpr (kPairs) {  // into the order of this lane's elements
      const uint32_t own0 = odd ? w[2] : w[0], own1 = odd ? w[3] : w[1];
      const uint32_t others0 = neighbours(odd ? w[0] : w[2]), others1 = neighbours(odd ? w[1] : w[3]);
      w = u32x4{odd ? others0 : own0, odd ? others1 : own1, odd ? own0 : others0, odd ? own1 : others1};
    }
#pragma unroll
    for (int v = 0; v < PARTS; ++v) {
      A f[VEC], r[VEC];
      LV::unpack(rx[v], f);
      if constexpr (RES) LV::unpack(rr[v], r);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const bool keep = kept(w, v * VEC + i, a.least);
        if constexpr (RES) f[i] = keep ? __builtin_elementwise_fma(f[i], scale, r[i]) : r[i];
        else f[i] = keep ? f[i] * scale : (A)0;
      }
      store_loose<LV>(y + place(v), LV::pack(f));
    }
    return;
  }
  const int64_t e0 = group * kGroup;
  if (e0 >= a.n) return;
  const u32x4 w = random_words((uint64_t)group, a.offset, seed);
#pragma unroll
  for (int i = 0; i < kGroup; ++i) {
    if (e0 + i >= a.n) break;
    using L1 = LaneVec<T, 1>;
    A f[1], r[1] = {0};
    L1::unpack(L1::load(x + e0 + i), f);
    if constexpr (RES) L1::unpack(L1::load(res + e0 + i), r);
    if constexpr (RES) f[0] = kept(w, i, a.least) ? __builtin_elementwise_fma(f[0], scale, r[0]) : r[0];
    else f[0] = kept(w, i, a.least) ? f[0] * scale : (A)0;
    L1::store(y + e0 + i, L1::pack(f));
  }
}

template <typename T> void launch_dropout(DropoutArgs a, hipStream_t stream) {
  constexpr int64_t per_block = (int64_t)kBlock * kGroup;
  const dim3 grid((unsigned)((a.n + per_block - 1) / per_block));
  if (a.residual) hipLaunchKernelGGL((dropout_kernel<T, true>), grid, dim3(kBlock), 0, stream, a);
  else hipLaunchKernelGGL((dropout_kernel<T, false>), grid, dim3(kBlock), 0, stream, a);
}

}  // namespace
}  // namespace gn

using namespace gn;

extern "C" int gnnhwc_dropout(const void *x, const void *residual, void *y, int64_t n, double p, uint64_t seed, const int64_t *seed_at,
                              uint64_t offset, int dtype, void *stream) {
  if (dtype != GN_F32 && dtype != GN_F64 && dtype != GN_F16 && dtype != GN_BF16)
    return fail(GNNHWC_ERR_INVALID_ARGUMENT, "unknown dtype code %d", dtype);
  if (!(p >= 0 && p <= 1)) return fail(GNNHWC_ERR_INVALID_ARGUMENT, "p must be 0 to 1");
  if (n < 0 || n > (int64_t)1 << 34) return fail(GNNHWC_ERR_INVALID_ARGUMENT, "size out of range: at most 2^34 elements");
  if (n == 0) return GNNHWC_OK;
  if (!x || !y) return fail(GNNHWC_ERR_INVALID_ARGUMENT, "null tensor");
  if ((uintptr_t)seed_at % 8) return fail(GNNHWC_ERR_INVALID_ARGUMENT, "seed_at must be aligned to 8 bytes");
  DropoutArgs a = {};
  a.x = x; a.residual = residual; a.y = y;
  a.n = n;
  a.seed_at = seed_at; a.seed = seed; a.offset = offset;
  a.least = (uint32_t)floor(p * 65536.0 + 0.5);
  a.scale = a.least < 65536 ? 65536.0 / (65536.0 - a.least) : 0.0;
  switch (dtype) {
    case GN_F32: launch_dropout<float>(a, (hipStream_t)stream); break;
    case GN_F64: launch_dropout<double>(a, (hipStream_t)stream); break;
    case GN_F16: launch_dropout<f16_t>(a, (hipStream_t)stream); break;
    default: launch_dropout<bf16_t>(a, (hipStream_t)stream); break;
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? GNNHWC_OK : fail(GNNHWC_ERR_LAUNCH, "gnnhwc_dropout: %s", hipGetErrorString(e));
}
