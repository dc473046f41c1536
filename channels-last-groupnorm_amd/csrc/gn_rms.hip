// Kernels of the root-mean-square norm (gn_rms.h) instantiated and launched for ONE element type, selected with
// -DGN_INST_DTYPE=0..3 (f32, f64, f16, bf16).
#include <type_traits>

#include "gn_rms.h"

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
constexpr int kVec = vec_of<elem_t>::value;
// Most lane vectors of a row of 1024 lanes.
constexpr int kWideVectors = kMostChannels / (sizeof(elem_t) == 8 ? 2 : 1) / (kVec * 1024);

// Calls f with the vectors of a lane and the threads of a workgroup as constants.
template <typename F> void with_width(const RowCut &cut, F &&f) {
  typedef std::integral_constant<int, 256> Narrow;
  typedef std::integral_constant<int, 1024> Wide;
  typedef std::integral_constant<int, 1> One;
  typedef std::integral_constant<int, 2> Two;
  typedef std::integral_constant<int, 3> Three;
  if (cut.threads <= 256) {
    if (cut.nv <= 1) return f(One(), Narrow());
    if (cut.nv == 2) return f(Two(), Narrow());
    return f(Three(), Narrow());
  }
  // rows longer than 256 lanes of three vectors hold
  if constexpr (kWideVectors > 2) {
    if (cut.nv == 3) return f(Three(), Wide());
    if (cut.nv > 3) return f(std::integral_constant<int, 4>(), Wide());
  }
  return f(Two(), Wide());
}

// ---- forward ----
template <typename P, int VEC, int NV, int THREADS, bool RAGGED, bool QUANT, bool STREAM>
void fwd_launch(const RmsFwd &a, const RowCut &cut, hipStream_t stream) {
  const int rows = cut.threads / cut.lpr;
  const dim3 grid((unsigned)((a.rows + rows - 1) / rows)), block(cut.threads);
  if (a.res) hipLaunchKernelGGL((rms_fwd_kernel<elem_t, P, VEC, NV, THREADS, RAGGED, true, QUANT, STREAM>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((rms_fwd_kernel<elem_t, P, VEC, NV, THREADS, RAGGED, false, QUANT, STREAM>), grid, block, 0, stream, a);
}
template <typename P, bool QUANT> void fwd_params(const RmsFwd &a, const RowCut &cut, hipStream_t stream) {
  const bool streams = a.rows * a.C * (int64_t)sizeof(elem_t) * (a.res ? 2 : 1) > kCachedBytes;
  if (cut.vec == 1) return fwd_launch<P, 1, 1, 256, false, QUANT, false>(a, cut, stream);
  with_width(cut, [&](auto nv, auto threads) {
    constexpr int NV = decltype(nv)::value, THREADS = decltype(threads)::value;
    if (cut.ragged) fwd_launch<P, kVec, NV, THREADS, true, QUANT, false>(a, cut, stream);
    else if (streams) fwd_launch<P, kVec, NV, THREADS, false, QUANT, true>(a, cut, stream);
    else fwd_launch<P, kVec, NV, THREADS, false, QUANT, false>(a, cut, stream);
  });
}

// ---- backward ----
template <typename P, int VEC, int NV, int THREADS, bool RAGGED, bool STREAM>
void bwd_launch(const RmsBwd &a, const RowCut &cut, hipStream_t stream, int blocks) {
  const int lanes = cut.lpr < 64 ? 64 : cut.lpr, groups = cut.threads / lanes;
  const size_t lds = (size_t)(groups / 2) * NV * VEC * lanes * sizeof(A);
  const dim3 grid((unsigned)blocks), block(cut.threads);
  if (a.ds) hipLaunchKernelGGL((rms_bwd_kernel<elem_t, P, VEC, NV, THREADS, RAGGED, true, STREAM>), grid, block, lds, stream, a);
  else hipLaunchKernelGGL((rms_bwd_kernel<elem_t, P, VEC, NV, THREADS, RAGGED, false, STREAM>), grid, block, lds, stream, a);
}
template <typename P> void bwd_params(const RmsBwd &a, const RowCut &cut, hipStream_t stream, int blocks) {
  const bool streams = a.rows * a.C * (int64_t)sizeof(elem_t) * (a.ds ? 3 : 2) > kCachedBytes;
  if (cut.vec == 1) return bwd_launch<P, 1, 1, 256, false, false>(a, cut, stream, blocks);
  with_width(cut, [&](auto nv, auto threads) {
    constexpr int NV = decltype(nv)::value, THREADS = decltype(threads)::value;
    if (cut.ragged) bwd_launch<P, kVec, NV, THREADS, true, false>(a, cut, stream, blocks);
    else if (streams) bwd_launch<P, kVec, NV, THREADS, false, true>(a, cut, stream, blocks);
    else bwd_launch<P, kVec, NV, THREADS, false, false>(a, cut, stream, blocks);
  });
}

}  // namespace

hipError_t GN_CAT(launch_rms_fwd_, GN_SUFFIX)(const RmsFwd &a, const RowCut &cut, int pdtype, bool quant, hipStream_t stream) {
#if GN_INST_DTYPE != 1
  if (quant) {
    if (pdtype == GN_INST_DTYPE) fwd_params<elem_t, true>(a, cut, stream);
    else fwd_params<wide_param_t, true>(a, cut, stream);
    return hipGetLastError();
  }
#endif
  if (pdtype == GN_INST_DTYPE) fwd_params<elem_t, false>(a, cut, stream);
  else fwd_params<wide_param_t, false>(a, cut, stream);
  return hipGetLastError();
}

hipError_t GN_CAT(launch_rms_bwd_, GN_SUFFIX)(const RmsBwd &a, const RowCut &cut, int pdtype, int blocks, void *dw, hipStream_t stream) {
  if (blocks == 0) {  // no rows: dw is zero
  } else if (pdtype == GN_INST_DTYPE) bwd_params<elem_t>(a, cut, stream, blocks);
  else bwd_params<wide_param_t>(a, cut, stream, blocks);
  if (dw) {
    const PartialSum p = {a.part, {dw, nullptr}, blocks, a.C, a.C, pdtype};
    hipLaunchKernelGGL((partial_sum_kernel<A>), dim3((unsigned)((a.C + kSumColumns - 1) / kSumColumns)), dim3(kSumThreads), 0, stream, p);
  }
  return hipGetLastError();
}

}  // namespace gn
