// The norm over many gradients and their clipping (see include/gnnhwc_tokens.h).
//
//   total = |s| sqrt(sum g^2),    out = g * (s min(1, max / (total + eps)))
// Two launches per table of tensors: partial sums, then the factor and the products.  Memory bounds both: 568 M bf16 gradients
// 190 us (6.0 TB/s), their products in float32 600 to 620 (5.5 to 5.7).  Workgroups take chunks of kClipChunk elements, neighbours
// in time neighbours in memory; the tensors' addresses travel as a kernel argument, so that nothing is copied to the device and no
// address is kept.  Every workgroup of the second pass adds all
// partial sums itself, in the same order, which costs it less than a launch in between would.
#include <math.h>
#include <stdint.h>
#include "gn_rms.h"

namespace gn {
namespace {

__device__ __forceinline__ const ClipEntry &entry_of(const ClipTable &t, unsigned chunk) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.e[mid].first_chunk <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return t.e[lo];
}

__device__ __forceinline__ double block_sum(double v, double *lds) {
  v = segment_sum(v, 64);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = lds[0] + lds[1] + lds[2] + lds[3];
  __syncthreads();
  return v;
}

// Squares are added in float64: those of large or tiny gradients leave the range of a float (and the additions hide behind the
// loads).
template <typename T> __device__ double chunk_squares(const T *p, int n) {
  constexpr int VEC = vec_of<T>::value;
  using LV = LaneVec<T, VEC>;
  using A = acc_of_t<T>;
  constexpr int kSteps = kClipChunk / (VEC * kBlock);
  double sum = 0;
  if (n == kClipChunk) {
    typename LV::raw_t r[kSteps];
#pragma unroll
    for (int k = 0; k < kSteps; ++k) r[k] = load_loose<LV>(p + (k * kBlock + (int)threadIdx.x) * VEC);
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      A v[VEC];
      LV::unpack(r[k], v);
#pragma unroll
      for (int i = 0; i < VEC; ++i) sum += (double)v[i] * (double)v[i];
    }
    return sum;
  }
  const int whole = n / VEC;
  for (int j = threadIdx.x; j < whole; j += kBlock) {
    A v[VEC];
    LV::unpack(load_loose<LV>(p + j * VEC), v);
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum += (double)v[i] * (double)v[i];
  }
  for (int i = whole * VEC + threadIdx.x; i < n; i += kBlock) {
    A v[1];
    LaneVec<T, 1>::unpack(LaneVec<T, 1>::load(p + i), v);
    sum += (double)v[0] * (double)v[0];
  }
  return sum;
}

__global__ __launch_bounds__(kBlock) void clip_norm_kernel(const ClipTable t, double *part) {
  __shared__ double lds[4];
  double sum = 0;
  for (unsigned c = blockIdx.x; c < t.chunks; c += gridDim.x) {
    const ClipEntry &e = entry_of(t, c);
    const int64_t at = (int64_t)(c - e.first_chunk) * kClipChunk;
    const int n = (int)(e.n - at < kClipChunk ? e.n - at : kClipChunk);
    switch (e.types & 0xff) {
      case GN_F32: sum += chunk_squares((const float *)e.in + at, n); break;
      case GN_F64: sum += chunk_squares((const double *)e.in + at, n); break;
      case GN_F16: sum += chunk_squares((const f16_t *)e.in + at, n); break;
      default: sum += chunk_squares((const bf16_t *)e.in + at, n); break;
    }
  }
  sum = block_sum(sum, lds);
  if (threadIdx.x == 0) store_global<double>(part + blockIdx.x, sum);
}

// One sum of many partial ones, in their place: for lists of more tables than kClipTables.
__global__ __launch_bounds__(kBlock) void clip_sum_kernel(double *part, int parts) {
  __shared__ double lds[4];
  double sum = 0;
#pragma unroll 8
  for (int i = threadIdx.x; i < parts; i += kBlock) sum += load_global<double>(part + i);
  sum = block_sum(sum, lds);
  if (threadIdx.x == 0) store_global<double>(part, sum);
}

template <bool STREAM, typename T, typename U> __device__ void chunk_scale(const T *p, U *o, int n, double factor) {
  constexpr int VT = vec_of<T>::value, VU = vec_of<U>::value, VEC = VT < VU ? VT : VU;
  using LV = LaneVec<T, VEC>;
  using LU = LaneVec<U, VEC>;
  using A = typename acc_of<T>::type;
  using B = typename acc_of<U>::type;
  // products in float64 only where one of the types is
  typedef decltype(A() * B()) M;
  const M f = (M)factor;
  constexpr int kSteps = kClipChunk / (VEC * kBlock) < 8 ? kClipChunk / (VEC * kBlock) : 8;
  const int whole = n / VEC;
  auto one = [&](typename LV::raw_t r, int j) {
    A v[VEC];
    B u[VEC];
    LV::unpack(r, v);
#pragma unroll
    for (int i = 0; i < VEC; ++i) u[i] = (B)((M)v[i] * f);
    store_loose<LU>(o + j * VEC, LU::pack(u));
  };
  if (n == kClipChunk) {
    for (int k0 = 0; k0 < kClipChunk / (VEC * kBlock); k0 += kSteps) {
      typename LV::raw_t r[kSteps];
#pragma unroll
      for (int k = 0; k < kSteps; ++k) r[k] = load_once<LV, STREAM>(p + ((k0 + k) * kBlock + (int)threadIdx.x) * VEC);
#pragma unroll
      for (int k = 0; k < kSteps; ++k) one(r[k], (k0 + k) * kBlock + (int)threadIdx.x);
    }
    return;
  }
  for (int j = threadIdx.x; j < whole; j += kBlock) one(load_loose<LV>(p + j * VEC), j);
  for (int i = whole * VEC + threadIdx.x; i < n; i += kBlock) {
    A v[1];
    B u[1];
    LaneVec<T, 1>::unpack(LaneVec<T, 1>::load(p + i), v);
    u[0] = (B)((M)v[0] * f);
    LaneVec<U, 1>::store(o + i, LaneVec<U, 1>::pack(u));
  }
}
template <bool STREAM, typename T> __device__ __forceinline__ void scale_to(const T *p, void *o, int64_t at, int n, double f, int type) {
  switch (type) {
    case GN_F32: chunk_scale<STREAM>(p, (float *)o + at, n, f); break;
    case GN_F64: chunk_scale<STREAM>(p, (double *)o + at, n, f); break;
    case GN_F16: chunk_scale<STREAM>(p, (f16_t *)o + at, n, f); break;
    default: chunk_scale<STREAM>(p, (bf16_t *)o + at, n, f); break;
  }
}

template <bool STREAM> __global__ __launch_bounds__(kBlock) void clip_apply_kernel(const ClipTable t, const ClipFinish q) {
  __shared__ double lds[4];
  double sum = 0;
  for (int i = threadIdx.x; i < q.parts; i += kBlock) sum += load_global<double>(q.part + i);
  sum = block_sum(sum, lds);
  const double scale = q.grad_scale < 0 ? -q.grad_scale : q.grad_scale;
  const double total = scale * __builtin_sqrt(sum);
  const double bound = q.max_norm == (double)INFINITY ? 1.0 : q.max_norm / (total + q.eps);
  const double factor = bound >= 1.0 ? q.grad_scale : q.grad_scale * bound;  // (a NaN stays one)
  if (blockIdx.x == 0 && threadIdx.x == 0 && q.total) store_scalar<double>(q.total, 0, q.total_dtype, total);
  if (q.in_place && factor == 1.0) return;
  // from the end: the first pass has left the last of a set larger than the memory-side cache there
  for (unsigned i = blockIdx.x; i < t.chunks; i += gridDim.x) {
    const unsigned c = t.chunks - 1 - i;
    const ClipEntry &e = entry_of(t, c);
    const int64_t at = (int64_t)(c - e.first_chunk) * kClipChunk;
    const int n = (int)(e.n - at < kClipChunk ? e.n - at : kClipChunk);
    const int to = e.types >> 8;
    switch (e.types & 0xff) {
      case GN_F32: scale_to<STREAM>((const float *)e.in + at, e.out, at, n, factor, to); break;
      case GN_F64: scale_to<STREAM>((const double *)e.in + at, e.out, at, n, factor, to); break;
      case GN_F16: scale_to<STREAM>((const f16_t *)e.in + at, e.out, at, n, factor, to); break;
      default: scale_to<STREAM>((const bf16_t *)e.in + at, e.out, at, n, factor, to); break;
    }
  }
}

}  // namespace

hipError_t launch_clip_norm(const ClipTable &t, double *part, int blocks, hipStream_t stream) {
  hipLaunchKernelGGL(clip_norm_kernel, dim3((unsigned)blocks), dim3(kBlock), 0, stream, t, part);
  return hipGetLastError();
}
hipError_t launch_clip_sum(double *part, int parts, hipStream_t stream) {
  hipLaunchKernelGGL(clip_sum_kernel, dim3(1), dim3(kBlock), 0, stream, part, parts);
  return hipGetLastError();
}
hipError_t launch_clip_apply(const ClipTable &t, const ClipFinish &f, bool streams, int blocks, hipStream_t stream) {
  if (streams) hipLaunchKernelGGL(clip_apply_kernel<true>, dim3((unsigned)blocks), dim3(kBlock), 0, stream, t, f);
  else hipLaunchKernelGGL(clip_apply_kernel<false>, dim3((unsigned)blocks), dim3(kBlock), 0, stream, t, f);
  return hipGetLastError();
}

}  // namespace gn
