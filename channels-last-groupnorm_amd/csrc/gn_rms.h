// Root-mean-square norm of rows, with the residual's addition in front and, optionally, 8-bit results with scales.
//
//   s = x + residual            (rounded to the data type once: s is a tensor of the residual stream)
//   y[c] = s[c] r w[c],         r = 1 / sqrt(mean_c s^2 + eps)
// backward, with g = dy w and h = s r:
//   dx = r (g - h mean_c(g h)) + ds,        dw[c] = sum over rows of dy h
// Quantised: per block of channels (or row) a = max |y|, scale = max(a / q_most, 2^-126), q = round(y / scale).
//
// What bounds them is memory: a row is read once, kept packed in registers between the sum of squares and the result, and
// written once: forward of float16 (65536, 2560) with its sum 219 us, 6.1 TB/s; bf16 (16384, 1280) 30.1 us, 5.6; in 8 bits with
// 128 channels a block bf16 (16384, 2560) 52.9 us, 5.6; a copy of their sizes runs at 5.7.  `lpr` lanes share a row (a power of
// two: part of a wavefront, or several wavefronts that add their sums through LDS), each with NV lane vectors, vector k of lane
// l being k * lpr + l, so that every access of a wavefront is one run of memory.
//
// A row whose length no lane vector divides ends with a vector that starts early enough to fit (RAGGED): its first elements
// are the previous vector's last ones, leave the sums, and are written twice with the same value.  Vectors are loaded and
// stored at the alignment of an element, which this hardware does in one access.
#pragma once
#include "gn_device.h"
#include "gn_tokens.h"

namespace gn {

template <typename R, int ALIGN> struct loose {
  typedef R type __attribute__((aligned(ALIGN)));
};
template <typename LV, typename T> __device__ __forceinline__ typename LV::raw_t load_loose(const T *p) {
  typedef typename loose<typename LV::raw_t, sizeof(T)>::type U;
  return *(const global_mem<U> *)p;
}
// STREAM: without a place in the caches, for tensors that no cache can hold until somebody reads them again.
template <typename LV, bool STREAM, typename T> __device__ __forceinline__ typename LV::raw_t load_once(const T *p) {
  typedef typename loose<typename LV::raw_t, sizeof(T)>::type U;
  if constexpr (STREAM) return __builtin_nontemporal_load((const global_mem<U> *)p);
  else return *(const global_mem<U> *)p;
}
template <typename LV, typename T> __device__ __forceinline__ void store_loose(T *p, typename LV::raw_t r) {
  typedef typename loose<typename LV::raw_t, sizeof(T)>::type U;
  __builtin_nontemporal_store((U)r, (global_mem<U> *)p);
}

template <typename T> using acc_of_t = typename acc_of<T>::type;
// y / d, where inv is 1 / d rounded: a product and one correction by its remainder (Markstein), which leaves the rounded quotient
// but for cases next to the middle of two floats.
__device__ __forceinline__ float quotient(float y, float d, float inv) {
  const float q = y * inv;
  return __builtin_fmaf(__builtin_fmaf(-q, d, y), inv, q);
}
// 1 / sqrt(ss / n + eps) of a row's sum of squares.  Whatever it is off by is off in all of the row, so that each of its steps is
// rounded once: the mean by quotient(), the root from the hardware's estimate (an ulp) and one Newton step in the form
// r + r (1 - v r^2) / 2, whose correction needs few bits.  About a dozen instructions, where a division, a root and a division
// take fifty; those are left for where the step would meet a zero, an infinity or a subnormal.
__device__ __forceinline__ float row_rstd(float ss, int n, double inv_n, double eps) {
  const float v = quotient(ss, (float)n, (float)inv_n) + (float)eps;
  if (v > 0x1p-100f && v < 0x1p+120f) {
    const float r = __builtin_amdgcn_rsqf(v), t = v * r;
    const float left = __builtin_fmaf(-t, r, 1.0f) - __builtin_fmaf(v, r, -t) * r;
    return __builtin_fmaf(0.5f * r, left, r);
  }
  return 1.0f / __builtin_sqrtf(ss / (float)n + (float)eps);
}
__device__ __forceinline__ double row_rstd(double ss, int n, double, double eps) { return 1.0 / __builtin_sqrt(ss / n + eps); }

// One lane vector's worth of VEC parameters of type P, as accumulators.
template <typename P, int VEC, typename A> __device__ __forceinline__ void load_params(const P *w, A (&v)[VEC]) {
  if constexpr (VEC == 1) {
    LaneVec<P, 1>::unpack(LaneVec<P, 1>::load(w), v);
  } else {
    constexpr int PV = vec_of<P>::value < VEC ? vec_of<P>::value : VEC;
    using LP = LaneVec<P, PV>;
#pragma unroll
    for (int i = 0; i < VEC; i += PV) {
      A t[PV];
      LP::unpack(load_loose<LP>(w + i), t);
#pragma unroll
      for (int j = 0; j < PV; ++j) v[i + j] = t[j];
    }
  }
}

// Which vectors of a row a lane holds.
template <int VEC, bool RAGGED> struct RowSlice {
  int lane, lpr, nvec, C;
  __device__ __forceinline__ int vector(int k) const { return k * lpr + lane; }
  __device__ __forceinline__ bool has(int k) const { return vector(k) < nvec; }
  // First element of vector k; lanes past the end take the last vector, whose memory is there.
  __device__ __forceinline__ int start(int k) const {
    int j = vector(k);
    j = j < nvec ? j : nvec - 1;
    const int e = j * VEC;
    return RAGGED ? (e + VEC <= C ? e : C - VEC) : e;
  }
  // Elements at the front of vector k that belong to the vector before.
  __device__ __forceinline__ int doubled(int k) const {
    if constexpr (!RAGGED) return 0;
    const int over = vector(k) * VEC + VEC - C;
    return over > 0 ? over : 0;
  }
};

// Sums of one or two values over the lanes of a row; all of them get the totals.  Rows of several wavefronts go through `lds`
// (two values per wavefront); `turn` alternates between two halves of it, so that one barrier per exchange is enough.
template <typename A> __device__ __forceinline__ void row_sum2(A &a, A &b, int lpr, A *lds, int turn) {
  if (lpr <= 64) {
    segment_sum2(a, b, lpr);
    return;
  }
  segment_sum2(a, b, 64);
  const int waves = lpr >> 6, wave = threadIdx.x >> 6, first = wave & ~(waves - 1);
  A *box = lds + turn * 32;
  if ((threadIdx.x & 63) == 0) {
    box[2 * wave] = a;
    box[2 * wave + 1] = b;
  }
  __syncthreads();
  a = b = (A)0;
  for (int i = 0; i < waves; ++i) {
    a += box[2 * (first + i)];
    b += box[2 * (first + i) + 1];
  }
}

// Largest magnitude, as the bits of a float: among them a NaN is the largest, so that it is not lost as in a maximum of floats.
__device__ __forceinline__ uint32_t magnitude_bits(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }
template <int CTRL> __device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
  const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xF, 0xF, false);
  return o > v ? o : v;
}
__device__ __forceinline__ uint32_t segment_max(uint32_t v, int width) {
  if (width >= 2) v = dpp_max<kDppQuadXor1>(v);
  if (width >= 4) v = dpp_max<kDppQuadXor2>(v);
  if (width >= 8) v = dpp_max<kDppRowHalfMirror>(v);
  if (width >= 16) v = dpp_max<kDppRowMirror>(v);
  for (int m = 16; m < 64; m <<= 1)
    if (width > m) {
      const uint32_t o = (uint32_t)__shfl_xor((int)v, m, 64);
      v = o > v ? o : v;
    }
  return v;
}
__device__ __forceinline__ uint32_t row_max(uint32_t v, int lpr, uint32_t *lds) {
  if (lpr <= 64) return segment_max(v, lpr);
  v = segment_max(v, 64);
  const int waves = lpr >> 6, wave = threadIdx.x >> 6, first = wave & ~(waves - 1);
  if ((threadIdx.x & 63) == 0) lds[wave] = v;
  __syncthreads();
  v = 0;
  for (int i = 0; i < waves; ++i) v = lds[first + i] > v ? lds[first + i] : v;
  return v;
}

// VEC values as 8-bit numbers, packed.  |v| <= q_most up to the rounding of the scale, which both conversions round down to
// q_most.
template <int VEC> struct Bytes {
  uint32_t w[(VEC + 3) / 4];
};
template <int VEC> __device__ __forceinline__ Bytes<VEC> pack_bytes(const float (&v)[VEC], int qtype) {
  Bytes<VEC> r;
#pragma unroll
  for (int i = 0; i < (VEC + 3) / 4; ++i) {
    float t[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) t[j] = 4 * i + j < VEC ? v[4 * i + j < VEC ? 4 * i + j : 0] : 0.0f;
    if (qtype == GN_F8) {
      int p = __builtin_amdgcn_cvt_pk_fp8_f32(t[0], t[1], 0, false);
      p = __builtin_amdgcn_cvt_pk_fp8_f32(t[2], t[3], p, true);
      r.w[i] = (uint32_t)p;
    } else {
      uint32_t p = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float n = t[j] == t[j] ? __builtin_rintf(t[j]) : 0.0f;  // a NaN shows in the scale
        p |= ((uint32_t)(int)n & 0xffu) << (8 * j);
      }
      r.w[i] = p;
    }
  }
  return r;
}

template <typename T, typename P, int VEC, int NV, int THREADS, bool RAGGED, bool RES, bool QUANT, bool STREAM>
__global__ __launch_bounds__(THREADS) void rms_fwd_kernel(const RmsFwd q) {
  using A = acc_of_t<T>;
  using LV = LaneVec<T, VEC>;
  typedef typename LV::raw_t raw_t;
  __shared__ A lds[64];
  __shared__ uint32_t lds_max[16];
  const RowSlice<VEC, RAGGED> cut = {(int)threadIdx.x & (q.lpr - 1), q.lpr, q.nvec, q.C};
  int64_t row = (int64_t)blockIdx.x * (blockDim.x >> q.lpr_log2) + (threadIdx.x >> q.lpr_log2);
  const bool live = row < q.rows;
  row = live ? row : q.rows - 1;  // lanes past the last row compute it too, and do not store

  const T *x = (const T *)q.x + row * q.x_stride;
  const T *res = RES ? (const T *)q.res + row * q.res_stride : nullptr;
  raw_t s[NV], r[RES ? NV : 1];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    s[k] = load_once<LV, STREAM>(x + cut.start(k));
    if constexpr (RES) r[k] = load_once<LV, STREAM>(res + cut.start(k));
  }
  // Asked for here, so that it is there when the sum is, and without a branch, at whose end the compiler would wait for all
  // that is on its way: without a weight P is T, and the row's own memory is read instead.
  const P *wp = q.w ? (const P *)q.w : (const P *)x;
  A w[NV][VEC];
#pragma unroll
  for (int k = 0; k < NV; ++k) load_params<P, VEC>(wp + cut.start(k), w[k]);
  A ss = 0, none = 0;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    A v[VEC];
    LV::unpack(s[k], v);
    if constexpr (RES) {
      A u[VEC];
      LV::unpack(r[k], u);
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] += u[i];
      s[k] = LV::pack(v);
      if (q.sum && live && cut.has(k)) store_loose<LV>((T *)q.sum + row * q.C + cut.start(k), s[k]);
      LV::unpack(s[k], v);
    }
    A part = 0;
#pragma unroll
    for (int i = 0; i < VEC; ++i) part += v[i] * v[i];
    if constexpr (RAGGED) {
      const int skip = cut.doubled(k);
      if (skip > 0) {  // one lane a row: a branch of its own is cheaper than a selection for every element of all
        issue_order_fence();
        part = 0;
#pragma unroll
        for (int i = 1; i < VEC; ++i) part += i >= skip ? v[i] * v[i] : (A)0;
      }
    }
    ss += cut.has(k) ? part : (A)0;
  }
  row_sum2(ss, none, q.lpr, lds, 0);
  const A rstd = row_rstd(ss, q.C, q.inv_c, q.eps);

  if constexpr (!QUANT) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      A v[VEC];
      LV::unpack(s[k], v);
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = q.w ? v[i] * rstd * w[k][i] : v[i] * rstd;
      if (live && cut.has(k)) store_loose<LV>((T *)q.y + row * q.C + cut.start(k), LV::pack(v));
    }
  } else {
    float y[NV][VEC];
    uint32_t most[NV], whole = 0;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      LV::unpack(s[k], y[k]);
      most[k] = 0;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        y[k][i] = q.w ? y[k][i] * rstd * w[k][i] : y[k][i] * rstd;
        const uint32_t b = magnitude_bits(y[k][i]);
        most[k] = b > most[k] ? b : most[k];
      }
      if constexpr (RAGGED) {
        const int skip = cut.doubled(k);
        if (skip > 0) {  // (the doubled elements may belong to another block)
          issue_order_fence();
          most[k] = 0;
#pragma unroll
          for (int i = 1; i < VEC; ++i) {
            const uint32_t b = i >= skip ? magnitude_bits(y[k][i]) : 0;
            most[k] = b > most[k] ? b : most[k];
          }
        }
      }
      if (!cut.has(k)) most[k] = 0;
      whole = most[k] > whole ? most[k] : whole;
    }
    if (q.block_lanes == 0) whole = row_max(whole, q.lpr, lds_max);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const uint32_t b = q.block_lanes == 0 ? whole : segment_max(most[k], q.block_lanes);
      const float a = __builtin_bit_cast(float, b) / q.q_most;
      const float scale = a < 0x1p-126f ? 0x1p-126f : a;  // (a NaN stays)
      // (against a product with inv alone bf16 (700000, 80) 39.5 -> 42 us, (16384, 2560) the same; divisions 55.6 and 53.3)
      const float inv = 1.0f / scale, divisor = inv > 0 ? scale : 0.0f;  // (an infinite scale has no remainders: y * 0 stays)
      if (!live || !cut.has(k)) continue;
      const int j = cut.vector(k);
      if (q.block_lanes == 0) {
        if (j == 0) store_global<float>(q.scales + row, scale);
      } else if ((j & (q.block_lanes - 1)) == 0) {
        store_global<float>(q.scales + row * q.nblocks + j / q.block_lanes, scale);
      }
      float v[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = quotient(y[k][i], divisor, inv);
      const Bytes<VEC> p = pack_bytes<VEC>(v, q.qtype);
      uint8_t *out = (uint8_t *)q.y + row * q.C + cut.start(k);
      const int skip = cut.doubled(k);
      if (VEC == 1 || (RAGGED && skip > 0)) {  // the doubled elements may belong to a block with another scale
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          if (i >= skip) store_global<uint8_t>(out + i, (uint8_t)(p.w[i / 4] >> (8 * (i % 4))));
      } else if constexpr (VEC >= 4) {
        typedef uint32_t words_t __attribute__((ext_vector_type(VEC / 4)));
        words_t u;
        if constexpr (VEC == 4) u = p.w[0];
        else
#pragma unroll
          for (int i = 0; i < VEC / 4; ++i) u[i] = p.w[i];
        typedef typename loose<words_t, 1>::type U;
        __builtin_nontemporal_store((U)u, (global_mem<U> *)out);
      }
    }
  }
}

// Backward: float16 (65536, 2560) with a gradient of the sum 233 us (5.8 TB/s), bf16 (16384, 1280) 34.9 (4.8).  A workgroup
// walks over rows and keeps its share of dw in registers, in a fixed order, and leaves one partial row of dw; partial_sum_kernel
// adds those.  r is computed again from s, whose sum of squares rides along with that of g s, so that the forward saves no
// statistics: with G = sum g s, mean(g h) = r G / C.  The second term is h (r mean(g h)), not s (r^3 G / C): r^3 leaves a float's
// range where r and the result are well inside.  (That is one product more an element and nothing in time; g - h mean(g h) times
// r would keep all g of the sums, and with them one workgroup per CU less.)
template <typename T, typename P, int VEC, int NV, int THREADS, bool RAGGED, bool DS, bool STREAM>
__global__ __launch_bounds__(THREADS) void rms_bwd_kernel(const RmsBwd q) {
  using A = acc_of_t<T>;
  using LV = LaneVec<T, VEC>;
  typedef typename LV::raw_t raw_t;
  __shared__ A lds[64];
  extern __shared__ char lds_dyn[];
  const RowSlice<VEC, RAGGED> cut = {(int)threadIdx.x & (q.lpr - 1), q.lpr, q.nvec, q.C};
  const int rows_per_step = blockDim.x >> q.lpr_log2, sub = threadIdx.x >> q.lpr_log2;
  A dw[NV][VEC], w[NV][VEC];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    if (q.w) load_params<P, VEC>((const P *)q.w + cut.start(k), w[k]);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      dw[k][i] = 0;
      if (!q.w) w[k][i] = (A)1;
    }
  }
  int turn = 0;
  // (the bound does not depend on the lane: all wavefronts meet at the same barriers)
  const int64_t stride = (int64_t)gridDim.x * rows_per_step;
  for (int64_t base = (int64_t)blockIdx.x * rows_per_step; base < q.rows; base += stride, turn ^= 1) {
    const bool live = base + sub < q.rows;
    const int64_t row = live ? base + sub : q.rows - 1;
    const T *sp = (const T *)q.s + row * q.s_stride, *dyp = (const T *)q.dy + row * q.dy_stride;
    const T *dsp = DS ? (const T *)q.ds + row * q.ds_stride : nullptr;
    raw_t s[NV], dy[NV], ds[DS ? NV : 1];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      s[k] = load_once<LV, STREAM>(sp + cut.start(k));
      dy[k] = load_once<LV, STREAM>(dyp + cut.start(k));
      if constexpr (DS) ds[k] = load_once<LV, STREAM>(dsp + cut.start(k));
    }
    A ss = 0, gs = 0;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      A sv[VEC], dv[VEC];
      LV::unpack(s[k], sv);
      LV::unpack(dy[k], dv);
      const int skip = cut.doubled(k);
      A p0 = 0, p1 = 0;
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (!RAGGED || i >= skip) {
          p0 += sv[i] * sv[i];
          p1 += dv[i] * w[k][i] * sv[i];
        }
      ss += cut.has(k) ? p0 : (A)0;
      gs += cut.has(k) ? p1 : (A)0;
    }
    row_sum2(ss, gs, q.lpr, lds, turn);
    const A r = row_rstd(ss, q.C, q.inv_c, q.eps);
    const A c = -(r * gs * (A)q.inv_c) * r;
    if (!live) continue;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      A sv[VEC], dv[VEC], dx[VEC];
      LV::unpack(s[k], sv);
      LV::unpack(dy[k], dv);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const A dr = dv[i] * r, h = sv[i] * r;
        dw[k][i] += dr * sv[i];
        dx[i] = dr * w[k][i] + h * c;
      }
      if constexpr (DS) {
        A u[VEC];
        LV::unpack(ds[k], u);
#pragma unroll
        for (int i = 0; i < VEC; ++i) dx[i] += u[i];
      }
      if (q.dx && cut.has(k)) store_loose<LV>((T *)q.dx + row * q.C + cut.start(k), LV::pack(dx));
    }
  }
  if (!q.part) return;
  // rows of one wavefront, then the wavefronts that hold the same channels, halves at a time
  for (int m = q.lpr; m < 64; m <<= 1)
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int i = 0; i < VEC; ++i) dw[k][i] += __shfl_xor(dw[k][i], m, 64);
  A *box = (A *)lds_dyn;
  const int lanes = q.lpr < 64 ? 64 : q.lpr;  // threads that hold different channels, or copies of them
  for (int half = (int)(blockDim.x / lanes) >> 1; half > 0; half >>= 1) {
    const int g = threadIdx.x / lanes, t = threadIdx.x & (lanes - 1);
    __syncthreads();
    if (g >= half && g < 2 * half)
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < VEC; ++i) box[((g - half) * NV * VEC + k * VEC + i) * lanes + t] = dw[k][i];
    __syncthreads();
    if (g < half)
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < VEC; ++i) dw[k][i] += box[(g * NV * VEC + k * VEC + i) * lanes + t];
  }
  if ((int)threadIdx.x < q.lpr) {
    A *out = (A *)q.part + (int64_t)blockIdx.x * q.C;
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (cut.has(k))
#pragma unroll
        for (int i = 0; i < VEC; ++i) store_global<A>(out + cut.start(k) + i, dw[k][i]);
  }
}

// Sums of `count` rows of C partial results, in a fixed order: kSumColumns columns a workgroup and as many threads a column as
// make a few loads each, all in flight at once.  512 rows of 1280 take 4.0 us, of 128 as well: the way of what other dies have
// just written, which neither more columns nor fewer threads shorten (256 threads with 32 loads each: 6.4).
constexpr int kSumColumns = 16, kSumThreads = 1024;
template <typename A> __global__ __launch_bounds__(kSumThreads) void partial_sum_kernel(const PartialSum q) {
  constexpr int kSubs = kSumThreads / kSumColumns;
  __shared__ A lds[kSumThreads / 64][kSumColumns];
  const int lane = threadIdx.x & (kSumColumns - 1), sub = threadIdx.x / kSumColumns, col = blockIdx.x * kSumColumns + lane;
  const A *p = (const A *)q.part + (col < q.C ? col : q.C - 1);
  A acc = 0;
#pragma unroll 8
  for (int i = sub; i < q.count; i += kSubs) acc += load_global<A>(p + (int64_t)i * q.C);
#pragma unroll
  for (int m = kSumColumns; m < 64; m <<= 1) acc += __shfl_xor(acc, m, 64);
  if ((threadIdx.x & 63) < kSumColumns) lds[threadIdx.x >> 6][lane] = acc;
  __syncthreads();
  if (sub != 0 || col >= q.C) return;
  acc = 0;
#pragma unroll
  for (int i = 0; i < kSumThreads / 64; ++i) acc += lds[i][lane];
  void *out = col < q.split ? q.out[0] : q.out[1];
  if (out) store_scalar<A>(out, col < q.split ? col : col - q.split, q.out_dtype, acc);
}

}  // namespace gn
