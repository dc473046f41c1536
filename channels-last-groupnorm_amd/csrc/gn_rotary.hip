// Kernels of the rotary positions (gn_rotary.h) instantiated and launched for ONE element type, selected with
// -DGN_INST_DTYPE=0..3 (f32, f64, f16, bf16).
#include "gn_rotary.h"

#ifndef GN_INST_DTYPE
#error "compile with -DGN_INST_DTYPE=<0|1|2|3>"
#endif

namespace gn {

#if GN_INST_DTYPE == 0
typedef float elem_t;
typedef float wide_param_t;
#define GN_SUFFIX f32
#elif GN_INST_DTYPE == 1
typedef double elem_t;
typedef double wide_param_t;
#define GN_SUFFIX f64
#elif GN_INST_DTYPE == 2
typedef f16_t elem_t;
typedef float wide_param_t;
#define GN_SUFFIX f16
#else
typedef bf16_t elem_t;
typedef float wide_param_t;
#define GN_SUFFIX bf16
#endif
#define GN_CAT2(a, b) a##b
#define GN_CAT(a, b) GN_CAT2(a, b)

namespace {

typedef acc_of_t<elem_t> A;

template <typename P, int S, bool NEAR, bool NORM> void launch_one(const RotaryArgs &a, hipStream_t stream) {
  const int per_block = kBlock >> a.lanes_log2;
  const dim3 grid((unsigned)(((int64_t)a.tokens * a.groups + per_block - 1) / per_block));
  const size_t lds = (size_t)a.span * (a.D / 2) * sizeof(SinCos<A>);
  // Heads that no cache can hold are read past the caches where either half of a head is whole lines of memory (float16 (46800,
  // 24 + 24 heads, 128): 203 -> 192 us); other halves share lines, which are then fetched twice (float32 (308142, 2 + 1, 96): 134 -> 169).
  if constexpr (S * sizeof(elem_t) == 16) {
    const int64_t bytes = (int64_t)a.tokens * (a.side[0].heads + a.side[1].heads) * a.D * sizeof(elem_t);
    if (bytes > kCachedBytes && a.D / 2 * sizeof(elem_t) % 128 == 0 && (NEAR || 2 * a.P == a.D)) {
      hipLaunchKernelGGL((rotary_kernel<elem_t, P, S, NEAR, NORM, true>), grid, dim3(kBlock), lds, stream, a);
      return;
    }
  }
  hipLaunchKernelGGL((rotary_kernel<elem_t, P, S, NEAR, NORM, false>), grid, dim3(kBlock), lds, stream, a);
}
template <typename P, int S, bool NEAR> void launch_bwd(const RotaryArgs &a, int blocks, hipStream_t stream) {
  const int per_block = kBlock >> a.lanes_log2;
  // the walk's two tables of angles, and after it the groups' sums
  const size_t tables = (size_t)2 * a.span * (a.D / 2) * sizeof(SinCos<A>);
  const size_t sums = (size_t)per_block * a.D * sizeof(A) + (size_t)per_block * sizeof(int);
  const size_t lds = tables > sums ? tables : sums;
  hipLaunchKernelGGL((rotary_norm_bwd_kernel<elem_t, P, S, NEAR>), dim3((unsigned)blocks), dim3(kBlock), lds, stream, a);
}
// Calls f<channels of a lane vector, near>() for the width that the plan chose.
template <typename F> void with_vec(int vec, bool near, F &&f) {
  auto go = [&](auto s) {
    if (near) f(s, std::true_type());
    else f(s, std::false_type());
  };
  if (vec == 1) return go(std::integral_constant<int, 1>());
#if GN_INST_DTYPE == 1
  return go(std::integral_constant<int, 2>());
#else
#if GN_INST_DTYPE >= 2
  if (vec == 8) return go(std::integral_constant<int, 8>());
#endif
  return go(std::integral_constant<int, 4>());
#endif
}

}  // namespace

hipError_t GN_CAT(launch_rotary_, GN_SUFFIX)(const RotaryArgs &a, int vec, bool near, bool norm, int pdtype, hipStream_t stream) {
  with_vec(vec, near, [&](auto s, auto n) {
    if (!norm) launch_one<elem_t, decltype(s)::value, decltype(n)::value, false>(a, stream);
    else if (pdtype == GN_INST_DTYPE) launch_one<elem_t, decltype(s)::value, decltype(n)::value, true>(a, stream);
    else launch_one<wide_param_t, decltype(s)::value, decltype(n)::value, true>(a, stream);
  });
  return hipGetLastError();
}

hipError_t GN_CAT(launch_rotary_norm_bwd_, GN_SUFFIX)(const RotaryArgs &a, int vec, bool near, int pdtype, int blocks, void *const (&dw)[2],
                                                       hipStream_t stream) {
  if (blocks > 0) with_vec(vec, near, [&](auto s, auto n) {  // (no tokens: the weights' gradients are zero)
    if (pdtype == GN_INST_DTYPE) launch_bwd<elem_t, decltype(s)::value, decltype(n)::value>(a, blocks, stream);
    else launch_bwd<wide_param_t, decltype(s)::value, decltype(n)::value>(a, blocks, stream);
  });
  if (dw[0] || dw[1]) {
    const PartialSum p = {a.part, {dw[0], dw[1]}, blocks, 2 * a.D, a.D, pdtype};
    hipLaunchKernelGGL((partial_sum_kernel<A>), dim3((unsigned)((2 * a.D + kSumColumns - 1) / kSumColumns)), dim3(kSumThreads), 0, stream, p);
  }
  return hipGetLastError();
}

}  // namespace gn
