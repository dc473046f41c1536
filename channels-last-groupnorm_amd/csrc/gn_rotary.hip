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

template <typename P, int S, bool NEAR, bool WHOLE, bool NORM> void launch_one(const RotaryArgs &a, hipStream_t stream) {
  const int per_block = kBlock >> a.lanes_log2;
  const dim3 grid((unsigned)(((int64_t)a.tokens * a.groups + per_block - 1) / per_block));
  const size_t lds = (size_t)a.span * (a.D / 2) * sizeof(SinCos<A>);
  // Heads that no cache can hold are read past the caches where each access is whole lines of memory (float16 (46800, 24 + 24
  // heads, 128): 203 -> 192 us; bf16 (74800, 24 + 24, 64): 162 -> 153); other halves share lines, which are then fetched twice
  // (float32 (308142, 2 + 1, 96): 127 -> 167; not so heads that are whole in an access, bf16 (46800, 24 + 24, 96): 149 -> 142), as
  // are heads that stand in for missing ones (float32 (500000, 2 + 1, 64): 128 -> 148).
  if constexpr (S * sizeof(elem_t) == 16) {
    const int heads = a.side[0].heads + a.side[1].heads;
    const int64_t bytes = (int64_t)a.tokens * heads * a.D * sizeof(elem_t);
    const bool lines = a.D / (WHOLE ? 1 : 2) * sizeof(elem_t) % 128 == 0 && (WHOLE || NEAR || 2 * a.P == a.D);
    if (bytes > kCachedBytes && lines && a.groups * kRotaryHeads <= 2 * heads) {
      hipLaunchKernelGGL((rotary_kernel<elem_t, P, S, NEAR, WHOLE, NORM, true>), grid, dim3(kBlock), lds, stream, a);
      return;
    }
  }
  hipLaunchKernelGGL((rotary_kernel<elem_t, P, S, NEAR, WHOLE, NORM, false>), grid, dim3(kBlock), lds, stream, a);
}
template <typename P, int S, bool NEAR, bool WHOLE> void launch_bwd(const RotaryArgs &a, int blocks, hipStream_t stream) {
  const int per_block = kBlock >> a.lanes_log2;
  // the walk's two tables of angles, and after it the groups' sums
  const size_t tables = (size_t)2 * a.span * (a.D / 2) * sizeof(SinCos<A>);
  const size_t sums = (size_t)per_block * a.D * sizeof(A) + (size_t)per_block * sizeof(int);
  const size_t lds = tables > sums ? tables : sums;
  hipLaunchKernelGGL((rotary_norm_bwd_kernel<elem_t, P, S, NEAR, WHOLE>), dim3((unsigned)blocks), dim3(kBlock), lds, stream, a);
}
// Calls f<channels of a lane vector, near, whole>() for what the plan chose.
template <bool BACKWARD, typename F> void with_cut(const RotaryCut &cut, F &&f) {
  auto go = [&](auto s) {
    if constexpr (sizeof(elem_t) == 2 && decltype(s)::value > 1)
      if (cut.near) return f(s, std::true_type(), std::true_type());
    if constexpr (sizeof(elem_t) == 2 && decltype(s)::value == 8 && !BACKWARD)
      if (cut.whole) return f(s, std::false_type(), std::true_type());
    if constexpr (sizeof(elem_t) != 2 || decltype(s)::value == 1)
      if (cut.near) return f(s, std::true_type(), std::false_type());
    f(s, std::false_type(), std::false_type());
  };
  if (cut.vec == 1) return go(std::integral_constant<int, 1>());
#if GN_INST_DTYPE == 1
  return go(std::integral_constant<int, 2>());
#else
#if GN_INST_DTYPE >= 2
  if (cut.vec == 8) return go(std::integral_constant<int, 8>());
#endif
  return go(std::integral_constant<int, 4>());
#endif
}

}  // namespace

hipError_t GN_CAT(launch_rotary_, GN_SUFFIX)(const RotaryArgs &a, const RotaryCut &cut, bool norm, int pdtype, hipStream_t stream) {
  with_cut<false>(cut, [&](auto s, auto n, auto w) {
    if (!norm) launch_one<elem_t, decltype(s)::value, decltype(n)::value, decltype(w)::value, false>(a, stream);
    else if (pdtype == GN_INST_DTYPE) launch_one<elem_t, decltype(s)::value, decltype(n)::value, decltype(w)::value, true>(a, stream);
    else launch_one<wide_param_t, decltype(s)::value, decltype(n)::value, decltype(w)::value, true>(a, stream);
  });
  return hipGetLastError();
}

hipError_t GN_CAT(launch_rotary_norm_bwd_, GN_SUFFIX)(const RotaryArgs &a, const RotaryCut &cut, int pdtype, int blocks, void *const (&dw)[2],
                                                       hipStream_t stream) {
  if (blocks > 0) with_cut<true>(cut, [&](auto s, auto n, auto w) {  // (no tokens: the weights' gradients are zero)
    if (pdtype == GN_INST_DTYPE) launch_bwd<elem_t, decltype(s)::value, decltype(n)::value, decltype(w)::value>(a, blocks, stream);
    else launch_bwd<wide_param_t, decltype(s)::value, decltype(n)::value, decltype(w)::value>(a, blocks, stream);
  });
  if (dw[0] || dw[1]) {
    const PartialSum p = {a.part, {dw[0], dw[1]}, blocks, 2 * a.D, a.D, pdtype};
    hipLaunchKernelGGL((partial_sum_kernel<A>), dim3((unsigned)((2 * a.D + kSumColumns - 1) / kSumColumns)), dim3(kSumThreads), 0, stream, p);
  }
  return hipGetLastError();
}

}  // namespace gn
