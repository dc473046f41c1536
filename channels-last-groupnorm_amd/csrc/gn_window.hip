// Kernels of the attention (gn_window.h) instantiated and launched for ONE element type, selected with -DGN_INST_DTYPE=0, 2 or 3
// (f32, f16, bf16).
#include "gn_window.h"

#ifndef GN_INST_DTYPE
#error "compile with -DGN_INST_DTYPE=<0|2|3>"
#endif

namespace gn {

#if GN_INST_DTYPE == 0
typedef float elem_t;
#define GN_SUFFIX f32
#elif GN_INST_DTYPE == 2
typedef f16_t elem_t;
#define GN_SUFFIX f16
#else
typedef bf16_t elem_t;
#define GN_SUFFIX bf16
#endif
#define GN_CAT2(a, b) a##b
#define GN_CAT(a, b) GN_CAT2(a, b)

namespace {

// Calls f with the width that a head of D channels is padded to.
template <typename F> void with_width(int D, F &&f) {
  switch (window_width(D)) {
    case 64: return f(std::integral_constant<int, 64>());
    case 96: return f(std::integral_constant<int, 96>());
    case 128: return f(std::integral_constant<int, 128>());
    default:
      if constexpr (sizeof(elem_t) == 2) {  // (float32: the plan takes heads of 128 at most)
        if (D <= 160) f(std::integral_constant<int, 160>());
        else f(std::integral_constant<int, 256>());
      }
  }
}
dim3 grid_of(int items) { return dim3((unsigned)((items + 7) / 8 * 8)); }
}  // namespace

hipError_t GN_CAT(launch_window_forward_, GN_SUFFIX)(const WindowArgs &a, bool few, hipStream_t stream) {
  auto launch = [&](auto w, auto fine) {
    constexpr int DP = decltype(w)::value;
    constexpr bool FINE = decltype(fine)::value;
    if (few) hipLaunchKernelGGL((window_few_kernel<elem_t, DP, FINE>), grid_of(a.items), dim3(64 * Few<elem_t, DP>::kWaves), 0, stream, a);
    else hipLaunchKernelGGL((window_forward_kernel<elem_t, DP, FINE>), grid_of(a.items), dim3(kBlock), 0, stream, a);
  };
  with_width(a.D, [&](auto w) {
    if constexpr (sizeof(elem_t) == 2) {
      if (a.fine) return launch(w, std::true_type());
    }
    launch(w, std::false_type());
  });
  if (a.splits > 1) {
    const Joining joining(a.D, a.splits);
    hipLaunchKernelGGL((window_join_kernel<elem_t>), dim3((unsigned)joining.blocks((int64_t)a.B * a.H * a.L)), dim3(kBlock), 0, stream, a, joining);
  }
  return hipGetLastError();
}

hipError_t GN_CAT(launch_window_backward_, GN_SUFFIX)(const WindowArgs &a, const WindowArgs &kv, const WindowArgs &sinks, hipStream_t stream) {
  with_width(a.D, [&](auto w) {
    constexpr int DP = decltype(w)::value;
    if (a.items) hipLaunchKernelGGL((window_dq_kernel<elem_t, DP>), grid_of(a.items), dim3(kBlock), 0, stream, a);
    if (a.items && a.splits > 1) {
      const int64_t rows = (int64_t)a.B * a.H * a.L;
      const Joining joining(a.D, a.splits);
      hipLaunchKernelGGL((window_dq_sum_kernel<elem_t>), dim3((unsigned)joining.blocks(rows)), dim3(kBlock), 0, stream, a, joining);
    }
    auto keys = [&](auto parts) {
      constexpr int P = decltype(parts)::value;
      hipLaunchKernelGGL((window_dkv_kernel<elem_t, DP, P>), grid_of(kv.items), dim3(kBlock), 0, stream, kv);
      if (sinks.items) hipLaunchKernelGGL((window_sink_kernel<elem_t, DP, P>), grid_of(sinks.items), dim3(64 * Few<elem_t, DP>::kWaves), 0, stream, sinks);
    };
    if constexpr (DP <= (sizeof(elem_t) == 2 ? 128 : 96)) {
      keys(std::integral_constant<int, 3>());
    } else {
      keys(std::integral_constant<int, 1>());
      keys(std::integral_constant<int, 2>());
    }
  });
  if (kv.shares > 1 || kv.sinks > 0) {
    WindowArgs sum = kv;
    const int64_t heads = (int64_t)kv.B * kv.K;
    const Joining of_sinks(kv.D, kv.sink_parts), of_others(kv.D, kv.shares);
    sum.sink_blocks = kv.sinks > 0 ? (int)of_sinks.blocks(heads * kv.sinks) : 0;
    const int64_t others = kv.shares > 1 ? of_others.blocks(heads * (kv.S - kv.sinks)) : 0;
    hipLaunchKernelGGL((window_sum_kernel<elem_t>), dim3((unsigned)(sum.sink_blocks + others)), dim3(kBlock), 0, stream, sum, of_sinks, of_others);
  }
  return hipGetLastError();
}

}  // namespace gn
