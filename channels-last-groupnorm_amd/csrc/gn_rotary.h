// Rotary positions with several axes, optionally behind a root-mean-square norm of each head.
//
//   (u, v) -> (u cos a - v sin a, u sin a + v cos a),    a = position[axis of the pair] * frequency[pair]
// backward (the turn is orthogonal): the gradient turned by -a; behind a norm, with d that gradient, h = t r and g = d w,
//   dt = r (g - h mean(g h)),        dw = sum over heads and tokens of d h
//
// Memory bounds them: q and k are read once and written once; angles come from a position and P frequencies per token and are
// not read from tables: float16 (46800 tokens, 24 + 24 heads, 128) 192 us, 6.0 TB/s (a copy: 5.7); bf16 (16384, 20 + 20, 64)
// with a norm 31.5 us, 5.3 (a copy of that size: 5.1), its backward 47, 5.4.  A group of lanes (a power of two) takes one head at
// a time, each lane one or two lane vectors of it; it turns every `groups`-th head of its token, so that one set of sines and
// cosines serves several heads and neighbouring groups read neighbouring memory.
#pragma once
#include "gn_rms.h"

namespace gn {

// sin and cos of pos * freq.  The product is carried as an exact pair of floats and turned into revolutions with 1 / (2 pi) as
// a pair, so that the reduction loses nothing however long the angle is; then polynomials in z^2 on an eighth of a revolution
// (fits at Chebyshev nodes, errors 2.5e-9 and 5e-11).  About 30 instructions, where a float sine of a long angle takes a loop.
__device__ __forceinline__ void angle_sincos(float pos, float freq, float &sn, float &cs) {
  float p = pos * freq;
  pin(p);  // (the products and the errors below must be the rounded ones')
  const float pl = __builtin_fmaf(pos, freq, -p);
  constexpr float kTurn = 0.15915494f, kTurnLow = (float)(0.15915494309189533577 - (double)0.15915494f);
  float t = p * kTurn;
  pin(t);
  const float low = __builtin_fmaf(p, kTurn, -t) + (p * kTurnLow + pl * kTurn);
  const float r = (t - __builtin_rintf(t)) + low;
  const float m = __builtin_rintf(4.0f * r);
  const float z = __builtin_fmaf(m, -0.25f, r), z2 = z * z;
  const float s = z * __builtin_fmaf(z2, __builtin_fmaf(z2, __builtin_fmaf(z2, -75.39976950f, 81.59250773f), -41.34166241f), 6.283185288f);
  const float c = __builtin_fmaf(z2, __builtin_fmaf(z2, __builtin_fmaf(z2, __builtin_fmaf(z2, 59.21866124f, -85.44280388f), 64.93931580f), -19.73920865f), 1.0f);
  const int quarter = (int)m;
  const float a = quarter & 1 ? c : s, b = quarter & 1 ? s : c;
  sn = quarter & 2 ? -a : a;
  cs = (quarter + 1) & 2 ? -b : b;
}
__device__ __forceinline__ void angle_sincos(double pos, double freq, double &sn, double &cs) {
  const double a = pos * freq;
  sn = sin(a);
  cs = cos(a);
}

// Position on one axis, without control flow: all types are read as one word, integers of 64 bits by their lower half.
__device__ __forceinline__ float position_at(const RotaryArgs &q, int64_t at) {
  const uint32_t word = load_global<uint32_t>((const uint32_t *)q.pos + (at << (q.pos_type == 1 ? 1 : 0)));
  return q.pos_type == 2 ? __builtin_bit_cast(float, word) : (float)(int32_t)word;
}

// Sine and cosine of all pairs of the tokens that a workgroup works on, in LDS: [token - first][pair].  Each is computed once a
// workgroup; lanes that compute those of their own pairs take more instructions for them than for turning four heads (the
// backward behind a norm, bf16 (16384, 20 + 20, 64): 60 us, then bound by instructions).
// Pairs behind the turning ones get the identity.
template <typename A> struct SinCos {
  A sn, cs;
};
template <typename A> __device__ __forceinline__ void fill_angles(const RotaryArgs &q, int first, int tokens, SinCos<A> *table) {
  const int half = q.D >> 1;
  for (int i = threadIdx.x; i < tokens * half; i += kBlock) {
    const int t = div_by(i, q.by_half), j = i - t * half;
    const int token = first + t < q.tokens ? first + t : q.tokens - 1;
    const int b = div_by(token, q.by_L), l = token - b * q.L;
    int axis = 0;
#pragma unroll
    for (int a = 0; a < 3; ++a) axis += j >= q.ends[a] ? 1 : 0;
    const int at = axis < q.axes ? axis : q.axes - 1;
    const float pos = position_at(q, (int64_t)b * q.pos_stride[0] + (int64_t)l * q.pos_stride[1] + at);
    const float f = load_global<float>(q.freq + (j < q.P ? j : q.P - 1));
    SinCos<A> v;
    angle_sincos((A)pos, (A)f, v.sn, v.cs);
    v.sn = j < q.P ? v.sn * (A)q.sign : (A)0;
    v.cs = j < q.P ? v.cs : (A)1;
    table[i] = v;
  }
}

// What one lane holds of a head: lane vectors of S channels, neighbouring lanes neighbouring vectors, so that one access of a
// group is one run of memory.
// - Two vectors: far pairs (j, j + P) have one from either half of the turning channels, near pairs (2j, 2j + 1) one from either
//   half of the head.  (Two near vectors behind each other read every line twice: float16 (46800, 24 + 24 heads, 128) 286 us.)
// - One vector (WHOLE), and the access is the whole head: near pairs lie inside it, far ones trade values with the lane that
//   holds the other half.  Halves that are not whole lines of memory made the stores write 16 to 25 % more than the heads.
// The host's plan (gn_tokens.hip) chooses, and says what each takes.
template <typename T, int S, bool NEAR, bool WHOLE> struct PairLane {
  using A = acc_of_t<T>;
  static constexpr int kVecs = WHOLE ? 1 : 2, kPairs = WHOLE && NEAR ? S / 2 : S, kWidth = kVecs * S;
  static constexpr bool kHalves = NEAR && S > 1 && !WHOLE;
  static constexpr bool kTrade = WHOLE && !NEAR;  // the other halves of the pairs are another lane's
  int j0, j1, at0, at1, P, other;
  bool first, turns; // j1: first pair of the second vector, where that has pairs of its own
  __device__ __forceinline__ PairLane(const RotaryArgs &q, int lane) : P(q.P) {
    const int v = lane < q.nvec ? lane : q.nvec - 1;  // spare lanes repeat the last vector and store nothing
    j1 = at1 = other = 0;
    first = turns = true;
    if constexpr (kTrade) {
      at0 = v * S;
      first = at0 < P;
      turns = at0 < 2 * P;  // (S divides P)
      j0 = first ? at0 : turns ? at0 - P : 0;
      const int partner = first ? at0 + P : turns ? at0 - P : at0;
      other = ((int)threadIdx.x - lane + partner / S) * 4;
    } else if constexpr (WHOLE) {
      j0 = v * (S / 2);
      at0 = v * S;
    } else if constexpr (kHalves) {
      j0 = v * (S / 2);
      j1 = (q.nvec + v) * (S / 2);
      at0 = 2 * j0;
      at1 = 2 * j1;
    } else {
      j0 = v * S;
      const bool far = !NEAR && j0 < P;  // (S divides P where pairs are far)
      at0 = far ? j0 : 2 * j0;
      at1 = far ? j0 + P : 2 * j0 + S;
    }
  }
  __device__ __forceinline__ int pair(int i) const { return kHalves && i >= S / 2 ? j1 + i - S / 2 : j0 + i; }
  __device__ __forceinline__ int at(int k) const { return k ? at1 : at0; }
  typedef typename LaneVec<T, S>::raw_t raw_t;
  __device__ __forceinline__ void angles(const SinCos<A> *row, A (&sn)[kPairs], A (&cs)[kPairs]) const {
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const SinCos<A> v = row[pair(i)];
      sn[i] = kTrade && first ? -v.sn : v.sn;
      cs[i] = v.cs;
    }
  }
  template <bool STREAM = false> __device__ __forceinline__ void load(const T *p, raw_t (&r)[kVecs]) const {
#pragma unroll
    for (int k = 0; k < kVecs; ++k) r[k] = load_once<LaneVec<T, S>, STREAM>(p + at(k));
  }
  __device__ __forceinline__ static void unpack(const raw_t (&r)[kVecs], A (&v)[kWidth]) {
    A t[S];
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      LaneVec<T, S>::unpack(r[k], t);
#pragma unroll
      for (int i = 0; i < S; ++i) v[k * S + i] = t[i];
    }
  }
  __device__ __forceinline__ void store(T *p, const A (&v)[kWidth]) const {
    A t[S];
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
#pragma unroll
      for (int i = 0; i < S; ++i) t[i] = v[k * S + i];
      store_loose<LaneVec<T, S>>(p + at(k), LaneVec<T, S>::pack(t));
    }
  }
  template <typename W> __device__ __forceinline__ void weights(const W *w, A (&v)[kWidth]) const {
    A t[S];
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      load_params<W, S>(w + at(k), t);
#pragma unroll
      for (int i = 0; i < S; ++i) v[k * S + i] = t[i];
    }
  }
  __device__ __forceinline__ void turn(A (&v)[kWidth], const A (&sn)[kPairs], const A (&cs)[kPairs], bool partial) const {
    A was[kWidth];
#pragma unroll
    for (int c = 0; c < kWidth; ++c) was[c] = v[c];
    if constexpr (kTrade) {
#pragma unroll
      for (int c = 0; c < kWidth; ++c) {
        const A o = __builtin_bit_cast(float, __builtin_amdgcn_ds_bpermute(other, __builtin_bit_cast(int, v[c])));
        v[c] = was[c] * cs[c] + o * sn[c];
        v[c] = turns ? v[c] : was[c];
      }
      return;
    } else {
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const int a = NEAR ? 2 * i : i, b = NEAR ? 2 * i + 1 : S + i;
      v[a] = was[a] * cs[i] - was[b] * sn[i];
      v[b] = was[a] * sn[i] + was[b] * cs[i];
    }
    // channels behind the pairs are taken back, not multiplied by one and zero: an infinity there stays one
    if (partial)
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        const int a = NEAR ? 2 * i : i, b = NEAR ? 2 * i + 1 : S + i;
        const bool keep = pair(i) >= P;
        v[a] = keep ? was[a] : v[a];
        v[b] = keep ? was[b] : v[b];
      }
    }
  }
};

// Heads of one token for one group of lanes.
struct HeadWalk {
  bool live;
  int token, which, first, step, count, b, l;  // which: 0 q, 1 k; heads first, first + step, ...
};
__device__ __forceinline__ HeadWalk head_walk(const RotaryArgs &q, int group) {
  HeadWalk w;
  w.live = group < q.tokens * q.groups;
  group = w.live ? group : q.tokens * q.groups - 1;  // (the last one again: its token is in the workgroup's span)
  w.token = div_by(group, q.by_groups);
  const int g = group - w.token * q.groups;
  w.which = g >= q.side[0].groups ? 1 : 0;
  w.first = w.which ? g - q.side[0].groups : g;
  w.step = w.which ? q.side[1].groups : q.side[0].groups;
  w.count = w.which ? q.side[1].heads : q.side[0].heads;
  w.b = div_by(w.token, q.by_L);
  w.l = w.token - w.b * q.L;
  return w;
}
// Tokens that a workgroup's groups belong to: at most span, and often one less.
__device__ __forceinline__ int tokens_of(const RotaryArgs &q, int start, int subs) {
  const int n = div_by(start + subs - 1, q.by_groups) - div_by(start, q.by_groups) + 1;
  return n < q.span ? n : q.span;
}
// q's or k's tensors, field by field: both are scalar loads of the argument block and a selection.
struct Side {
  const void *in, *grad, *weight;
  void *out;
  int64_t in_stride[3], grad_stride[3], out_stride[3];
};
__device__ __forceinline__ Side side_of(const RotaryArgs &q, int which) {
  const RotarySide &a = q.side[0], &b = q.side[1];
  Side s;
  s.in = which ? b.in : a.in;
  s.grad = which ? b.grad : a.grad;
  s.weight = which ? b.weight : a.weight;
  s.out = which ? b.out : a.out;
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    s.in_stride[i] = which ? b.in_stride[i] : a.in_stride[i];
    s.grad_stride[i] = which ? b.grad_stride[i] : a.grad_stride[i];
    s.out_stride[i] = which ? b.out_stride[i] : a.out_stride[i];
  }
  return s;
}
__device__ __forceinline__ int64_t head_at(const int64_t (&s)[3], int b, int l) { return b * s[0] + l * s[1]; }

template <typename T, typename P, int S, bool NEAR, bool WHOLE, bool NORM, bool STREAM>
__global__ __launch_bounds__(kBlock) void rotary_kernel(const RotaryArgs q) {
  using A = acc_of_t<T>;
  using Lane = PairLane<T, S, NEAR, WHOLE>;
  constexpr int kHeads = kRotaryHeads;
  extern __shared__ char lds_dyn[];
  SinCos<A> *const table = (SinCos<A> *)lds_dyn;
  const int lane = threadIdx.x & (q.lanes - 1), sub = threadIdx.x >> q.lanes_log2, subs = kBlock >> q.lanes_log2;
  const int start = (int)blockIdx.x * subs;
  const HeadWalk walk = head_walk(q, start + sub);
  const Lane pl(q, lane);
  const Side side = side_of(q, walk.which);
  const bool stores = walk.live && lane < q.nvec, partial = 2 * q.P < q.D;
  const T *in = (const T *)side.in + head_at(side.in_stride, walk.b, walk.l);
  T *out = (T *)side.out + head_at(side.out_stride, walk.b, walk.l);
  const int64_t in_head = side.in_stride[2], out_head = side.out_stride[2];
  // all heads are asked for first and are on their way while the angles are computed
  typename Lane::raw_t r[kHeads][Lane::kVecs];
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const int h = walk.first + i * walk.step;
    pl.template load<STREAM>(in + (h < walk.count ? h : walk.first) * in_head, r[i]);
  }
  A sn[Lane::kPairs], cs[Lane::kPairs], w[Lane::kWidth];
  if constexpr (NORM) pl.weights((const P *)side.weight, w);
  const int first = div_by(start, q.by_groups);
  fill_angles(q, first, tokens_of(q, start, subs), table);
  __syncthreads();
  pl.angles(table + (walk.token - first) * (q.D >> 1), sn, cs);
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const int h = walk.first + i * walk.step;
    if (h >= walk.count) continue;
    A v[Lane::kWidth];
    pl.unpack(r[i], v);
    if constexpr (NORM) {
      A ss = 0;
#pragma unroll
      for (int c = 0; c < Lane::kWidth; ++c) ss += v[c] * v[c];
      ss = segment_sum(lane < q.nvec ? ss : (A)0, q.lanes);
      const A rstd = row_rstd(ss, q.D, q.inv_d, q.eps);
#pragma unroll
      for (int c = 0; c < Lane::kWidth; ++c) v[c] = v[c] * rstd * w[c];
    }
    pl.turn(v, sn, cs, partial);
    if (stores) pl.store(out + h * out_head, v);
  }
}

// Backward behind a norm: four lane vectors of q or k and four of their gradients at once (bf16 (16384, 20 + 20, 64): eight take
// the registers of a third workgroup a CU, 64 us instead of 50 with far pairs; two take 51 instead of 47 with near ones).  A group
// keeps its place among the heads (and so q or k) while it walks over tokens, and its share of dw in registers; a workgroup
// leaves one partial row of 2 D values (q's, k's).
template <typename T, typename P, int S, bool NEAR, bool WHOLE>
__global__ __launch_bounds__(kBlock) void rotary_norm_bwd_kernel(const RotaryArgs q) {
  using A = acc_of_t<T>;
  using Lane = PairLane<T, S, NEAR, WHOLE>;
  constexpr int kHeads = kRotaryBwdVecs / Lane::kVecs, kWidth = Lane::kWidth;
  extern __shared__ char lds_dyn[];
  const int lane = threadIdx.x & (q.lanes - 1), sub = threadIdx.x >> q.lanes_log2, subs = kBlock >> q.lanes_log2;
  const Lane pl(q, lane);
  const bool partial = 2 * q.P < q.D;
  const int start = (int)blockIdx.x * subs;
  const bool works = start + sub < q.walkers;  // (groups that do not fill a whole set of heads stay idle)
  const HeadWalk walk = head_walk(q, works ? start + sub : start);
  const Side side = side_of(q, walk.which);
  SinCos<A> *const tables = (SinCos<A> *)lds_dyn;
  const int first = div_by(start, q.by_groups), tokens = tokens_of(q, start, subs), half = q.D >> 1;
  A w[kWidth], dw[kWidth];
  pl.weights((const P *)side.weight, w);
#pragma unroll
  for (int c = 0; c < kWidth; ++c) dw[c] = 0;
  int turn = 0;
  // (the bound is the workgroup's: all wavefronts meet at the same barriers; two tables in turn, so that one is enough)
  for (int at = 0; first + at < q.tokens; at += q.token_step, turn ^= 1) {
    const bool there = works && walk.token + at < q.tokens;
    const int token = there ? walk.token + at : q.tokens - 1, b = div_by(token, q.by_L), l = token - b * q.L;
    const T *in = (const T *)side.in + head_at(side.in_stride, b, l), *grad = (const T *)side.grad + head_at(side.grad_stride, b, l);
    T *out = (T *)side.out + head_at(side.out_stride, b, l);
    typename Lane::raw_t rt[kHeads][Lane::kVecs], rd[kHeads][Lane::kVecs];
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      const int h = walk.first + i * walk.step < walk.count ? walk.first + i * walk.step : walk.first;
      pl.load(in + h * side.in_stride[2], rt[i]);
      pl.load(grad + h * side.grad_stride[2], rd[i]);
    }
    SinCos<A> *const table = tables + turn * q.span * half;
    fill_angles(q, first + at, tokens, table);
    __syncthreads();
    A sn[Lane::kPairs], cs[Lane::kPairs];
    pl.angles(table + (walk.token - first) * half, sn, cs);
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      const int h = walk.first + i * walk.step;
      if (!there || h >= walk.count) continue;
      A t[kWidth], d[kWidth], ss = 0, gt = 0;
      pl.unpack(rt[i], t);
      pl.unpack(rd[i], d);
      pl.turn(d, sn, cs, partial);
#pragma unroll
      for (int c = 0; c < kWidth; ++c) {
        ss += t[c] * t[c];
        gt += d[c] * w[c] * t[c];
      }
      if (lane >= q.nvec) ss = gt = 0;
      segment_sum2(ss, gt, q.lanes);
      // dt = r g - h (r mean(g h)) with mean(g h) = r gt / D, as in rms_bwd_kernel: r^3 would leave a float's range
      const A r = row_rstd(ss, q.D, q.inv_d, q.eps), m = -(r * gt * (A)q.inv_d) * r;
#pragma unroll
      for (int c = 0; c < kWidth; ++c) {
        const A dr = d[c] * r, h = t[c] * r;
        dw[c] += dr * t[c];
        d[c] = dr * w[c] + h * m;
      }
      if (lane < q.nvec) pl.store(out + h * side.out_stride[2], d);
    }
  }
  __syncthreads();
  // the workgroup's groups, q's and k's apart
  A *box = (A *)lds_dyn;  // [subs][D]
  int *kind = (int *)(box + subs * q.D);
  if (lane < q.nvec)
#pragma unroll
    for (int c = 0; c < kWidth; ++c) box[sub * q.D + pl.at(c / S) + c % S] = dw[c];
  if (lane == 0) kind[sub] = works ? walk.which : 2;
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * q.D; i += kBlock) {
    const int which = i >= q.D ? 1 : 0, c = i - which * q.D;
    A acc = 0;
    for (int g = 0; g < subs; ++g) acc += kind[g] == which ? box[g * q.D + c] : (A)0;
    store_global<A>((A *)q.part + (int64_t)blockIdx.x * 2 * q.D + i, acc);
  }
}

}  // namespace gn
