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
  if (D <= 64) f(std::integral_constant<int, 64>());
  else if (D <= 96) f(std::integral_constant<int, 96>());
  else if (D <= 128) f(std::integral_constant<int, 128>());
  else f(std::integral_constant<int, 256>());
}
dim3 grid_of(int items) { return dim3((unsigned)((items + 7) / 8 * 8)); }

}  // namespace

hipError_t GN_CAT(launch_window_forward_, GN_SUFFIX)(const WindowArgs &a, hipStream_t stream) {
  with_width(a.D, [&](auto w) { hipLaunchKernelGGL((window_forward_kernel<elem_t, decltype(w)::value>), grid_of(a.items), dim3(kBlock), 0, stream, a); });
  return hipGetLastError();
}

hipError_t GN_CAT(launch_window_few_, GN_SUFFIX)(const WindowArgs &a, hipStream_t stream) {
  with_width(a.D, [&](auto w) {
    constexpr int DP = decltype(w)::value;
    hipLaunchKernelGGL((window_few_kernel<elem_t, DP>), grid_of(a.items), dim3(64 * Few<elem_t, DP>::kWaves), 0, stream, a);
  });
  if (a.splits > 1) {
    const int64_t rows = (int64_t)a.B * a.H * a.L;
    hipLaunchKernelGGL((window_join_kernel<elem_t>), dim3((unsigned)((rows + 3) / 4)), dim3(kBlock), 0, stream, a);
  }
  return hipGetLastError();
}

hipError_t GN_CAT(launch_window_backward_, GN_SUFFIX)(const WindowArgs &a, const WindowArgs &kv, hipStream_t stream) {
  with_width(a.D, [&](auto w) {
    constexpr int DP = decltype(w)::value;
    if (a.items) hipLaunchKernelGGL((window_dq_kernel<elem_t, DP>), grid_of(a.items), dim3(kBlock), 0, stream, a);
    if constexpr (DP <= 128) {
      hipLaunchKernelGGL((window_dkv_kernel<elem_t, DP, 3>), grid_of(kv.items), dim3(kBlock), 0, stream, kv);
    } else {
      hipLaunchKernelGGL((window_dkv_kernel<elem_t, DP, 1>), grid_of(kv.items), dim3(kBlock), 0, stream, kv);
      hipLaunchKernelGGL((window_dkv_kernel<elem_t, DP, 2>), grid_of(kv.items), dim3(kBlock), 0, stream, kv);
    }
  });
  if (kv.shares > 1 || kv.sink_shares > 1) {
    const int64_t tiles = (kv.shares > 1 ? kv.tiles : kv.sink_tiles) - (kv.sink_shares > 1 ? 0 : kv.sink_tiles);
    const int64_t rows = (int64_t)kv.B * kv.K * tiles * kQueries;
    if (rows > 0) hipLaunchKernelGGL((window_sum_kernel<elem_t>), dim3((unsigned)((rows + 3) / 4)), dim3(kBlock), 0, stream, kv);
  }
  return hipGetLastError();
}

}  // namespace gn
