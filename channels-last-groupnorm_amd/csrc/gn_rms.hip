// Kernels of the root-mean-square norm (gn_rms.h) instantiated and launched for ONE element type, selected with
// -DGN_INST_DTYPE=0..3 (f32, f64, f16, bf16).
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

// ---- forward ----
template <typename P, int VEC, int NV, int THREADS, bool RAGGED, bool QUANT>
void fwd_launch(const RmsFwd &a, hipStream_t stream, unsigned grid, int threads) {
  if (a.res) hipLaunchKernelGGL((rms_fwd_kernel<elem_t, P, VEC, NV, THREADS, RAGGED, true, QUANT>), dim3(grid), dim3(threads), 0, stream, a);
  else hipLaunchKernelGGL((rms_fwd_kernel<elem_t, P, VEC, NV, THREADS, RAGGED, false, QUANT>), dim3(grid), dim3(threads), 0, stream, a);
}
template <typename P, bool RAGGED, bool QUANT> void fwd_width(const RmsFwd &a, const RowCut &cut, hipStream_t stream, unsigned grid) {
  if (cut.vec == 1) return fwd_launch<P, 1, 1, 256, false, QUANT>(a, stream, grid, cut.threads);
  if (cut.threads > 256) {
    if (cut.nv == 1) return fwd_launch<P, kVec, 1, 1024, RAGGED, QUANT>(a, stream, grid, cut.threads);
    if (kWideVectors < 3 || cut.nv == 2) return fwd_launch<P, kVec, 2, 1024, RAGGED, QUANT>(a, stream, grid, cut.threads);
    if constexpr (kWideVectors >= 3) {
      if (cut.nv == 3) return fwd_launch<P, kVec, 3, 1024, RAGGED, QUANT>(a, stream, grid, cut.threads);
      return fwd_launch<P, kVec, 4, 1024, RAGGED, QUANT>(a, stream, grid, cut.threads);
    }
  }
  switch (cut.nv) {
    case 1: return fwd_launch<P, kVec, 1, 256, RAGGED, QUANT>(a, stream, grid, cut.threads);
    case 2: return fwd_launch<P, kVec, 2, 256, RAGGED, QUANT>(a, stream, grid, cut.threads);
    case 3: return fwd_launch<P, kVec, 3, 256, RAGGED, QUANT>(a, stream, grid, cut.threads);
    case 4: return fwd_launch<P, kVec, 4, 256, RAGGED, QUANT>(a, stream, grid, cut.threads);
    case 5: return fwd_launch<P, kVec, 5, 256, RAGGED, QUANT>(a, stream, grid, cut.threads);
    case 6: return fwd_launch<P, kVec, 6, 256, RAGGED, QUANT>(a, stream, grid, cut.threads);
    default: return fwd_launch<P, kVec, 8, 256, RAGGED, QUANT>(a, stream, grid, cut.threads);
  }
}
template <typename P, bool QUANT> void fwd_params(const RmsFwd &a, const RowCut &cut, hipStream_t stream) {
  const int rows = cut.threads / cut.lpr;
  const unsigned grid = (unsigned)((a.rows + rows - 1) / rows);
  if (cut.ragged) fwd_width<P, true, QUANT>(a, cut, stream, grid);
  else fwd_width<P, false, QUANT>(a, cut, stream, grid);
}

// ---- backward ----
template <typename P, int VEC, int NV, int THREADS, bool RAGGED>
void bwd_launch(const RmsBwd &a, hipStream_t stream, unsigned grid, const RowCut &cut) {
  const int lanes = cut.lpr < 64 ? 64 : cut.lpr, groups = cut.threads / lanes;
  const size_t lds = (size_t)(groups / 2) * NV * VEC * lanes * sizeof(A);
  if (a.ds) hipLaunchKernelGGL((rms_bwd_kernel<elem_t, P, VEC, NV, THREADS, RAGGED, true>), dim3(grid), dim3(cut.threads), lds, stream, a);
  else hipLaunchKernelGGL((rms_bwd_kernel<elem_t, P, VEC, NV, THREADS, RAGGED, false>), dim3(grid), dim3(cut.threads), lds, stream, a);
}
template <typename P, bool RAGGED> void bwd_width(const RmsBwd &a, const RowCut &cut, hipStream_t stream, unsigned grid) {
  if (cut.vec == 1) return bwd_launch<P, 1, 1, 256, false>(a, stream, grid, cut);
  if (cut.threads > 256) {
    if (cut.nv == 1) return bwd_launch<P, kVec, 1, 1024, RAGGED>(a, stream, grid, cut);
    if (kWideVectors < 3 || cut.nv == 2) return bwd_launch<P, kVec, 2, 1024, RAGGED>(a, stream, grid, cut);
    if constexpr (kWideVectors >= 3) {
      if (cut.nv == 3) return bwd_launch<P, kVec, 3, 1024, RAGGED>(a, stream, grid, cut);
      return bwd_launch<P, kVec, 4, 1024, RAGGED>(a, stream, grid, cut);
    }
  }
  switch (cut.nv) {
    case 1: return bwd_launch<P, kVec, 1, 256, RAGGED>(a, stream, grid, cut);
    case 2: return bwd_launch<P, kVec, 2, 256, RAGGED>(a, stream, grid, cut);
    case 3: return bwd_launch<P, kVec, 3, 256, RAGGED>(a, stream, grid, cut);
    default: return bwd_launch<P, kVec, 4, 256, RAGGED>(a, stream, grid, cut);
  }
}
template <typename P> void bwd_params(const RmsBwd &a, const RowCut &cut, hipStream_t stream, unsigned grid) {
  if (cut.ragged) bwd_width<P, true>(a, cut, stream, grid);
  else bwd_width<P, false>(a, cut, stream, grid);
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
  } else if (pdtype == GN_INST_DTYPE) bwd_params<elem_t>(a, cut, stream, (unsigned)blocks);
  else bwd_params<wide_param_t>(a, cut, stream, (unsigned)blocks);
  if (dw) {
    const PartialSum p = {a.part, dw, blocks, a.C, pdtype, a.C};
    hipLaunchKernelGGL((partial_sum_kernel<A>), dim3((unsigned)((a.C + 15) / 16)), dim3(256), 0, stream, p);
  }
  return hipGetLastError();
}

}  // namespace gn
