// Softmax attention in which a token sees a window around it and a few first tokens (sinks): forward and backward.
//
//   s[i][j] = scale q[i] . k[j],   P[i][.] = softmax of s[i][.] over the tokens that i sees,   o[i] = sum_j P[i][j] v[j]
// backward, with delta[i] = do[i] . o[i] and dS[i][j] = P[i][j] (do[i] . v[j] - delta[i]):
//   dq[i] = scale sum_j dS[i][j] k[j],   dk[j] = scale sum_i dS[i][j] q[i],   dv[j] = sum_i P[i][j] do[i]
//
// Every product runs on matrix instructions of 32 x 32 x 16 whose result has one token of one side per lane, so that no value
// of a score tile changes lanes: S^T = K Q^T leaves a query in each lane's column, with 16 of 32 keys, and the second product
// takes them as its B operand where they are, for the order of its 16 summands is free as long as both operands have the same:
// summand i of half h is row 8 (i / 4) + 4 h + i % 4, which is also what a transposing read of two times four rows delivers.
// The running maximum and sum of the softmax then belong to a lane.
//
// Tiles of the other side are copied from memory into shared memory without passing through registers, two deep: the next one
// travels while this one is multiplied.  A row of a tile is cut into chunks of 16 bytes whose order depends on the row
// (chunk_of), so that rows read side by side lie in different banks.
#pragma once
#include <type_traits>
#include "gn_device.h"
#include "gn_window_args.h"

namespace gn {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x8_t __attribute__((ext_vector_type(8)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef short s16x8_t __attribute__((ext_vector_type(8)));

// Eight elements of a lane: an operand's share of 16 summands.
template <typename T> struct Operand;
template <> struct Operand<bf16_t> {
  typedef bf16x8_t type;
  static __device__ __forceinline__ f32x16_t product(type a, type b, f32x16_t c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Operand<f16_t> {
  typedef f16x8_t type;
  static __device__ __forceinline__ f32x16_t product(type a, type b, f32x16_t c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <> struct Operand<float> {  // eight products of two summands each
  typedef f32x8_t type;
  static __device__ __forceinline__ f32x16_t product(type a, type b, f32x16_t c) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
    return c;
  }
};
template <typename T> using operand_t = typename Operand<T>::type;
// Values 8 t .. 8 t + 7 of a lane's column, rounded to T once: what the products' results cost beside float32 operands, half a
// unit in the last place of each summand, like the operands that come from memory.
template <typename T> __device__ __forceinline__ operand_t<T> operand_of(const f32x16_t &v, int t) {
  if constexpr (sizeof(T) == 4) {
    f32x8_t r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = v[8 * t + i];
    return r;
  } else if constexpr (__is_same(T, bf16_t)) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = pack_bf16x2(v[8 * t + 2 * i], v[8 * t + 2 * i + 1]);
    return __builtin_bit_cast(bf16x8_t, r);
  } else {
    f16x8_t r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = (_Float16)v[8 * t + i];
    return r;
  }
}
__device__ __forceinline__ f32x16_t zeros16() {
  f32x16_t v;
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = 0.0f;
  return v;
}
// Row of a result tile that register r of a lane in half h holds.
__device__ __forceinline__ constexpr int row_of(int r, int h) { return 8 * (r / 4) + 4 * h + r % 4; }

template <typename T> __device__ __forceinline__ float to_float(const T *p) {
  float v[1];
  LaneVec<T, 1>::unpack(LaneVec<T, 1>::load(p), v);
  return v[0];
}

// ---- tiles in shared memory ----
template <typename T, int DP> struct Tile {
  static constexpr int kRows = sizeof(T) == 2 ? 64 : 32;
  static constexpr int kChunks = DP * (int)sizeof(T) / 16;  // of a row
  static constexpr int kBytes = kRows * kChunks * 16;

  // Place of chunk c in its row: four neighbouring rows lie in different quarters of the 64 banks, which suits the transposing
  // reads of four rows, and sixteen in different places, which suits the reads of a chunk of many rows.
  static __device__ __forceinline__ int chunk_of(int row, int c) {
    if constexpr (kChunks % 16 == 0) return c ^ ((row & 3) << 2 | (row >> 2 & 3));
    else if constexpr (kChunks % 8 == 0) return c ^ ((row >> 1 & 1) << 2 | (row >> 2 & 3));
    else return c ^ (row >> 2 & 3);
  }
};

// Where a lane finds its operands in a tile, the same for every tile and every 32 (columns: 16) rows of it: offsets that a constant
// is added to.  (The bits that a chunk's number and the row's pattern have are xor-ed: each step of channels costs a register, not
// an addition.)
template <typename T, int DP> struct LaneOffsets {
  using G = Tile<T, DP>;
  static constexpr int kRowBytes = G::kChunks * 16;
  // Wide heads keep one step's offsets and make the others of them: the steps' bits are the rows' to neither side.
  static constexpr bool kCompact = DP * (int)sizeof(T) >= 512;
  static_assert(!kCompact || (kRowBytes & (kRowBytes - 1)) == 0, "a row's bytes are a power of two");
  static constexpr int kSteps = kCompact ? 1 : DP / 16, kParts = kCompact ? 1 : DP / 32;
  int rows[sizeof(T) == 2 ? 1 : 2][kSteps], columns[kParts][sizeof(T) == 2 ? 2 : 8];
  int steps;
  // Whether step x of a product over a head's channels has any of them.  (16 bits: a step past the head costs less than to ask)
  __device__ __forceinline__ bool has(int x) const {
    if constexpr (sizeof(T) == 2) return true;
    else return x == 0 || x < steps;
  }
  static __device__ __forceinline__ int step_of(int first, int x, int bytes) {
    pin(first);  // (or they would all be made ahead of the loop, and kept)
    return first ^ x * bytes;
  }
  __device__ __forceinline__ int row_offset(int i, int x) const {
    if constexpr (kCompact) return step_of(rows[i][0], x, 16 * (int)sizeof(T));
    else return rows[i][x];
  }
  __device__ __forceinline__ int column_offset(int x, int i) const {
    if constexpr (kCompact) return step_of(columns[0][i], x, 32 * (int)sizeof(T));
    else return columns[x][i];
  }
  __device__ __forceinline__ void init(int D) {
    steps = (D + 15) / 16;
    const int lane = threadIdx.x & 63, h = lane >> 5, row = lane & 31;
#pragma unroll
    for (int x = 0; x < kSteps; ++x) {
      if constexpr (sizeof(T) == 2) {
        rows[0][x] = row * kRowBytes + G::chunk_of(row, 2 * x + h) * 16;
      } else {
        rows[0][x] = row * kRowBytes + G::chunk_of(row, 4 * x + 2 * h) * 16;
        rows[1][x] = row * kRowBytes + G::chunk_of(row, 4 * x + 2 * h + 1) * 16;
      }
    }
#pragma unroll
    for (int x = 0; x < kParts; ++x) {
      if constexpr (sizeof(T) == 2) {
        // a group of 16 lanes reads four rows of 16 channels, four to a lane, and each lane is left with a channel
        const int m = lane & 15, r = 4 * h + (m >> 2), chunk = 4 * x + (lane >> 4 & 1) * 2 + (m >> 1 & 1);
#pragma unroll
        for (int i = 0; i < 2; ++i) columns[x][i] = (r + 8 * i) * kRowBytes + G::chunk_of(r + 8 * i, chunk) * 16 + (m & 1) * 8;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) columns[x][i] = row_of(i, h) * kRowBytes + G::chunk_of(row_of(i, h), (32 * x + row) >> 2) * 16 + (row & 3) * 4;
      }
    }
  }
  // Operand whose rows are the tile's rows FIRST .. FIRST + 31 (a multiple of 32), summands 16 x + 8 h ..
  template <int FIRST> __device__ __forceinline__ operand_t<T> of_rows(const char *tile, int x) const {
    if constexpr (sizeof(T) == 2) {
      return *(const operand_t<T> *)(tile + row_offset(0, x) + FIRST * kRowBytes);
    } else {
      const f32x4 a = *(const f32x4 *)(tile + row_offset(0, x) + FIRST * kRowBytes), b = *(const f32x4 *)(tile + row_offset(1, x) + FIRST * kRowBytes);
      return f32x8_t{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    }
  }
  // Operand whose rows are the channels 32 x .., its summands the tile's rows FIRST .. FIRST + 15 in a result's order.
  template <int FIRST> __device__ __forceinline__ operand_t<T> of_columns(char *tile, int x) const {
    if constexpr (sizeof(T) == 2) {
      typedef __attribute__((address_space(3))) s16x4_t lds4;
      const s16x4_t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *)(tile + column_offset(x, 0) + FIRST * kRowBytes));
      const s16x4_t b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *)(tile + column_offset(x, 1) + FIRST * kRowBytes));
      return __builtin_bit_cast(operand_t<T>, s16x8_t{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]});
    } else {
      f32x8_t r;
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i] = *(const float *)(tile + column_offset(x, i) + FIRST * kRowBytes);
      return r;
    }
  }
};

template <typename P> __device__ __forceinline__ P *uniform(P *p) {
  const uint64_t v = (uint64_t)p;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)v), hi = __builtin_amdgcn_readfirstlane((int)(v >> 32));
  return (P *)((uint64_t)hi << 32 | lo);
}

// Each lane's BYTES from memory (base + offset) into shared memory, the lanes' behind each other from `to` on; base and `to` are the same
// for all of them.  (The compiler would have every transposing read wait for all copies that are on their way, other buffers'
// too: it is not told of these.  Nothing is written to a register but m0, which nothing else here uses; tiles_turn waits.)
template <int BYTES> __device__ __forceinline__ void copy_to_lds(const char *base, unsigned offset, unsigned to) {
  to = __builtin_amdgcn_readfirstlane(to);
  base = uniform(base);
  if constexpr (BYTES == 16)
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %2" ::"v"(offset), "s"(to), "s"(base) : "memory");
  else
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, %2" ::"v"(offset), "s"(to), "s"(base) : "memory");
}
__device__ __forceinline__ unsigned lds_address(const void *p) { return (unsigned)(uintptr_t)(const __attribute__((address_space(3))) void *)p; }

// Copies tiles of ROWS rows into shared memory, by LANES lanes.  Rows past `last` and chunks past the head are other rows and chunks
// of the same tensor (memory that is there, and values whose products are left out).
template <typename T, int DP, int ROWS, int LANES> struct TileCopy {
  using G = Tile<T, DP>;
  static constexpr int kCopies = ROWS * G::kChunks / LANES;
  static_assert(ROWS * G::kChunks % LANES == 0, "a tile is whole copies");
  unsigned offset[kCopies];
  int stride;
  // row and chunk of copy i of this lane; `lane` may hide that they are constants
  static __device__ __forceinline__ int row_at(int i, int lane) { return (i * LANES + lane) / G::kChunks; }
  static __device__ __forceinline__ int byte_at(int i, int lane, int D) {
    const int slot = i * LANES + lane, c = G::chunk_of(slot / G::kChunks, slot % G::kChunks) * 16;  // (its own inverse)
    return c < D * (int)sizeof(T) ? c : 0;
  }
  __device__ __forceinline__ void init(int D, int token_bytes) {
    stride = token_bytes;
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const int lane = threadIdx.x % LANES;
      offset[i] = (unsigned)row_at(i, lane) * (unsigned)stride + byte_at(i, lane, D);
    }
  }
  // from: the tile's first row; left: its last row, counted from there; `to`: where the tile goes, plus 1024 times the wavefront's
  // number among those that copy it.
  __device__ __forceinline__ void issue(const char *from, int left, unsigned to, int D) const {
    if (left >= ROWS - 1) {
#pragma unroll
      for (int i = 0; i < kCopies; ++i) copy_to_lds<16>(from, offset[i], to + i * LANES * 16);
    } else {
      int lane = threadIdx.x % LANES;
      pin(lane);  // (so that nothing of this lies in registers all along)
#pragma unroll
      for (int i = 0; i < kCopies; ++i) {
        const int r = row_at(i, lane);
        copy_to_lds<16>(from, (unsigned)(r < left ? r : left) * (unsigned)stride + byte_at(i, lane, D), to + i * LANES * 16);
      }
    }
  }
};
// Two tensors' tiles at once, one walk's after the other: the places in memory move on by additions.
template <typename T, int DP, int ROWS, int LANES> struct TilePair {
  TileCopy<T, DP, ROWS, LANES> x, y;
  const char *at_x, *at_y;
  int last, D, first;  // last row, the next tile's first
  __device__ __forceinline__ void init(int D_, int x_bytes, int y_bytes, int last_) {
    D = D_;
    last = last_;
    x.init(D_, x_bytes);
    y.init(D_, y_bytes);
  }
  __device__ __forceinline__ void go_to(const char *base_x, const char *base_y, int row) {
    first = row;
    at_x = uniform(base_x + (int64_t)row * x.stride);
    at_y = uniform(base_y + (int64_t)row * y.stride);
  }
  __device__ __forceinline__ void issue(unsigned to, unsigned apart) const {
    x.issue(at_x, last - first, to, D);
    y.issue(at_y, last - first, to + apart, D);
  }
  __device__ __forceinline__ void advance(int tiles) {
    first += tiles * ROWS;
    at_x += (int64_t)tiles * ROWS * x.stride;
    at_y += (int64_t)tiles * ROWS * y.stride;
  }
};
// All of this workgroup's copies have arrived and all of its reads of shared memory are done.
__device__ __forceinline__ void tiles_turn() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// ---- which tokens see which ----
// A sample's tokens: keys 0 .. n - 1; query i stands at place i + off, those with first <= i < last stand among the keys.
struct Sample {
  int n, off, first, last;
};
__device__ __forceinline__ Sample sample_of(const WindowArgs &a, int b) {
  Sample s;
  s.n = a.S;
  if (a.lengths) {
    const int64_t n = a.length_type ? load_global<int64_t>((const int64_t *)a.lengths + b) : (int64_t)load_global<int>((const int *)a.lengths + b);
    s.n = __builtin_amdgcn_readfirstlane(n < 0 ? 0 : n < a.S ? (int)n : a.S);  // (all that a workgroup does by it is scalar)
  }
  s.off = (a.at_end ? s.n : a.S) - a.L;
  s.first = s.off < 0 ? -s.off : 0;
  s.last = s.n - s.off < a.L ? s.n - s.off : a.L;
  return s;
}
// What a query sees: keys low .. low + count - 1, and keys below `sinks`.
struct Sight {
  int low, count, sinks;
  __device__ __forceinline__ bool sees(int j) const { return (unsigned)(j - low) < (unsigned)count || j < sinks; }
};
__device__ __forceinline__ Sight sight_of(const WindowArgs &a, const Sample &s, int i) {
  Sight g = {0, 0, 0};
  if (i >= s.first && i < s.last) {
    const int p = i + s.off, high = p + a.right < s.n ? p + a.right : s.n - 1;
    g.low = p > a.left ? p - a.left : 0;
    g.count = high - g.low + 1;
    g.sinks = a.sinks < s.n ? a.sinks : s.n;
    if (a.causal && p + 1 < g.sinks) g.sinks = p + 1;
  }
  return g;
}
// The places from which a key is seen: from, .. from + count - 1 (the queries that are there).
struct Seen {
  int from, count;
};
__device__ __forceinline__ Seen seen_of(const WindowArgs &a, const Sample &s, int j) {
  Seen g = {0, 0};
  if (j < s.n && s.last > s.first) {
    int lo = j - a.right, hi = j + a.left;
    if (j < a.sinks) {  // by all
      if (!a.causal) lo = 0;
      hi = s.n - 1;
    }
    const int least = s.first + s.off, most = s.last - 1 + s.off;
    lo = lo > least ? lo : least;
    hi = hi < most ? hi : most;
    g.from = lo;
    g.count = hi < lo ? 0 : hi - lo + 1;
  }
  return g;
}
// Tiles of `rows` keys that a workgroup with queries at places low .. high has to visit: those of the sinks, then the window's.
struct Walk {
  int sinks, first, last;  // tiles of the sinks; the window's tiles behind them: first .. last
};
__device__ __forceinline__ Walk walk_of(const WindowArgs &a, const Sample &s, int low, int high, int rows) {
  Walk w;
  int sinks = a.sinks < s.n ? a.sinks : s.n;
  if (a.causal && high + 1 < sinks) sinks = high + 1;
  w.sinks = (sinks + rows - 1) / rows;
  const int from = low > a.left ? low - a.left : 0, to = high + a.right < s.n ? high + a.right : s.n - 1;
  w.first = from / rows;
  if (w.first < w.sinks) w.first = w.sinks;
  w.last = to / rows;
  return w;
}

__device__ __forceinline__ int rest_by(int n, const Divisor &v) { return n - div_by(n, v) * v.d; }

// The work of this workgroup, of a.items ordered by key head; a.items and beyond: none.  Workgroups are dealt to the eight dies in
// turn, each with a cache of its own that a head's keys and values are to be in once: heads are dealt to the dies in turn, or, where
// they do not come out even, each die has a stretch of the work, or, where samples have lengths that would make those uneven, all
// is dealt in turn.  (training: 2 x 4096 tokens, 24 heads over 8 of 128, 535 us by heads or stretches, 590 in turn; 3 x 4096, padded,
// 9 over 3, 475 us in turn, 760 by stretches)
__device__ __forceinline__ int work_item(const WindowArgs &a) {
  const int id = blockIdx.x, die = id & 7, n = id >> 3;
  if (a.order == kHeadsInTurn) return (div_by(n, a.by_per_head) * 8 + die) * a.per_head + rest_by(n, a.by_per_head);
  return a.order == kStretches ? die * ((a.items + 7) >> 3) + n : id;
}

// The kernel's arguments, read again behind a loop, so that those of the results take no registers in it.
__device__ __forceinline__ const WindowArgs &arguments_again() {
  auto p = (const __attribute__((address_space(4))) WindowArgs *)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const WindowArgs *)p;
}

// ---- rows by their formulas, for results that are not finite ----
// A tile's products reach over all of its rows: what a token does not see has the weight 0 there, and 0 times an infinity or a NaN
// of such a token is NaN.  A row that comes out infinite or NaN is therefore computed again over the pairs that see each other
// alone, by one wavefront, in float32.  Rows that have to be NaN whatever they see (their own q is not finite: so are all scores,
// and infinite ones differ by NaN) are seen to be at once: a training that has diverged has nothing but those.  A walk ends where all
// that it adds up has become NaN, which nothing behind it changes: float16 gradients of a loss that was scaled too far are NaN as a
// rule, while q, k and v are finite (4 x 4112 tokens, 20 heads of 64, window 512, all of the gradient NaN: 7 ms, 101 to the end).
template <typename T> __device__ __forceinline__ float dot(const T *a, const T *b, int D) {
  float s = 0.0f;
#pragma unroll 4
  for (int d = 0; d < D; ++d) s = __builtin_fmaf(to_float(a + d), to_float(b + d), s);
  return s;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int m = 32; m; m >>= 1) v = fmaxf(v, __shfl_xor(v, m));
  return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int m = 32; m; m >>= 1) v += __shfl_xor(v, m);
  return v;
}
// Calls f(j0, j) for the keys that a query sees, 64 at a time: j of this lane, or -1.  Ends where f returns true.
template <typename F> __device__ __forceinline__ void for_keys(const Sight &g, F &&f) {
  const int lane = threadIdx.x & 63;
  const int sinks = g.count > 0 && g.low < g.sinks ? g.low : g.sinks;  // (those of the window once)
  for (int j0 = 0; j0 < sinks; j0 += 64)
    if (f(j0, j0 + lane < sinks ? j0 + lane : -1)) return;
  for (int j0 = g.low; j0 < g.low + g.count; j0 += 64)
    if (f(j0, j0 + lane < g.low + g.count ? j0 + lane : -1)) return;
  if (g.count > 0 && g.low + g.count < g.sinks)
    for (int j0 = g.low + g.count; j0 < g.sinks; j0 += 64)
      if (f(j0, j0 + lane < g.sinks ? j0 + lane : -1)) return;
}
// Whether a row of D channels holds a NaN, or with `infinite` anything that is not finite; all lanes of a wavefront ask together.
template <typename T> __device__ __forceinline__ bool holds_nan(const T *p, int D, bool infinite) {
  const int lane = threadIdx.x & 63;
  bool bad = false;
  for (int d = lane; d < D; d += 64) {
    const float v = to_float(p + d);
    bad = bad || (infinite ? !(v * 0.0f == 0.0f) : v != v);
  }
  return __any(bad);
}
// A row's sums, channels lane, lane + 64, .. of a lane each; those past the head, which are left alone, are NaN.
__device__ __forceinline__ void clear_row(float (&acc)[4], int D) {
#pragma unroll
  for (int x = 0; x < 4; ++x) acc[x] = x * 64 + (int)(threadIdx.x & 63) < D ? 0.0f : __builtin_nanf("");
}
// Whether all of them are NaN (a maximum is, if both of its operands are).
__device__ __forceinline__ bool all_nan(const float (&acc)[4]) {
  const float most = fmaxf(fmaxf(acc[0], acc[1]), fmaxf(acc[2], acc[3]));
  return __all(most != most);
}
template <typename T> __device__ __forceinline__ void fill_nan(T *p, int D) {
  const float t[1] = {__builtin_nanf("")};
  for (int d = threadIdx.x & 63; d < D; d += 64) LaneVec<T, 1>::store(p + d, LaneVec<T, 1>::pack(t));
}
// Channels d .. d + N - 1 of a row of out, rounded, and what the rounding left.  (The backward's delta, the sum of do * out, is made
// of both: dP - delta of a token that sees a few others is a small difference, and 2^-9 of out is not small against it.)
template <typename T, int N> __device__ __forceinline__ void store_out(const WindowArgs &a, int b, int h, int i, int d, const float (&t)[N]) {
  using LV = LaneVec<T, N>;
  const auto raw = LV::pack(t);
  LV::store((T *)a.out.row(b, i, h) + d, raw);
  if constexpr (sizeof(T) == 2) {
    if (a.rest) {
      float r[N];
      LV::unpack(raw, r);
#pragma unroll
      for (int e = 0; e < N; ++e) r[e] = t[e] - r[e];
      LV::store((T *)a.rest + (((int64_t)b * a.L + i) * a.H + h) * a.D + d, LV::pack(r));
    }
  }
}
template <typename T> __device__ void row_again(const WindowArgs &a, const Sample &s, int b, int h, int i) {
  const int lane = threadIdx.x & 63, kh = div_by(h, a.by_group);
  const Sight g = sight_of(a, s, i);
  const T *q = (const T *)a.q.row(b, i, h);
  float most = -INFINITY;
  bool nan = holds_nan(q, a.D, true);  // (so is the sum, and all of the row, where a score is NaN or +infinity)
  if (!nan)
    for_keys(g, [&](int, int j) {
      const float v = j >= 0 ? dot(q, (const T *)a.k.row(b, j, kh), a.D) * a.scale_log2 : -INFINITY;
      most = fmaxf(most, v);
      nan = __any(!(v < INFINITY));
      return nan;
    });
  if (nan) {
    fill_nan((T *)a.out.row(b, i, h), a.D);
    if (a.lse && lane == 0) store_global<float>(a.lse + ((int64_t)b * a.H + h) * a.L + i, __builtin_nanf(""));
    return;
  }
  most = wave_max(most);
  most = most == -INFINITY ? 0.0f : most;
  float sum = 0.0f;
  for_keys(g, [&](int, int j) {
    if (j >= 0) sum += __builtin_amdgcn_exp2f(dot(q, (const T *)a.k.row(b, j, kh), a.D) * a.scale_log2 - most);
    return false;
  });
  sum = wave_sum(sum);
  float o[4];
  clear_row(o, a.D);
  for_keys(g, [&](int j0, int j) {
    const float p = j >= 0 ? __builtin_amdgcn_exp2f(dot(q, (const T *)a.k.row(b, j, kh), a.D) * a.scale_log2 - most) / sum : 0.0f;
    for (int u = 0; u < 64; ++u) {
      const int ju = __shfl(j, u);
      const float pu = __shfl(p, u);
      if (ju < 0) break;
      const T *v = (const T *)a.v.row(b, ju, kh);
#pragma unroll
      for (int x = 0; x < 4; ++x)
        if (x * 64 + lane < a.D) o[x] = __builtin_fmaf(pu, to_float(v + x * 64 + lane), o[x]);
    }
    return all_nan(o);
  });
#pragma unroll
  for (int x = 0; x < 4; ++x)
    if (x * 64 + lane < a.D) {
      const float t[1] = {o[x]};
      store_out<T, 1>(a, b, h, i, x * 64 + lane, t);
    }
  if (a.lse && lane == 0) store_global<float>(a.lse + ((int64_t)b * a.H + h) * a.L + i, most + __builtin_amdgcn_logf(sum));
}
// dq of one row.
template <typename T> __device__ void dq_again(const WindowArgs &a, const Sample &s, int b, int h, int i, float lse, float delta) {
  const int lane = threadIdx.x & 63, kh = div_by(h, a.by_group);
  const T *q = (const T *)a.q.row(b, i, h), *g = (const T *)a.dout.row(b, i, h);
  if (lse != lse || delta != delta) return fill_nan((T *)a.dq.row(b, i, h), a.D);
  float acc[4];
  clear_row(acc, a.D);
  for_keys(sight_of(a, s, i), [&](int, int j) {
    float ds = 0.0f;
    if (j >= 0) {
      const float p = __builtin_amdgcn_exp2f(dot(q, (const T *)a.k.row(b, j, kh), a.D) * a.scale_log2 - lse);
      ds = p * (dot(g, (const T *)a.v.row(b, j, kh), a.D) - delta);
    }
    for (int u = 0; u < 64; ++u) {
      const int ju = __shfl(j, u);
      const float du = __shfl(ds, u);
      if (ju < 0) break;
      const T *k = (const T *)a.k.row(b, ju, kh);
#pragma unroll
      for (int x = 0; x < 4; ++x)
        if (x * 64 + lane < a.D) acc[x] = __builtin_fmaf(du, to_float(k + x * 64 + lane), acc[x]);
    }
    return all_nan(acc);
  });
  T *to = (T *)a.dq.row(b, i, h);
#pragma unroll
  for (int x = 0; x < 4; ++x)
    if (x * 64 + lane < a.D) {
      const float t[1] = {acc[x] * a.scale};
      LaneVec<T, 1>::store(to + x * 64 + lane, LaneVec<T, 1>::pack(t));
    }
}
// dk or dv of one row.
template <typename T> __device__ void dkv_again(const WindowArgs &a, const Sample &s, int b, int kh, int j, bool of_k) {
  const int lane = threadIdx.x & 63;
  const T *k = (const T *)a.k.row(b, j, kh), *v = (const T *)a.v.row(b, j, kh);
  const Seen w = seen_of(a, s, j);
  if (holds_nan(k, a.D, false) || (of_k && holds_nan(v, a.D, false))) return fill_nan((T *)(of_k ? a.dk.row(b, j, kh) : a.dv.row(b, j, kh)), a.D);
  float acc[4];
  clear_row(acc, a.D);
  bool nan = false;
  for (int h = kh * a.group; h < (kh + 1) * a.group && !nan; ++h) {
    const int64_t rows = ((int64_t)b * a.H + h) * a.L;
    for (int i0 = 0; i0 < w.count && !nan; i0 += 64) {
      const int i = i0 + lane < w.count ? w.from + i0 + lane - s.off : -1;
      float t = 0.0f;
      if (i >= 0) {
        t = __builtin_amdgcn_exp2f(dot((const T *)a.q.row(b, i, h), k, a.D) * a.scale_log2 - load_global<float>(a.lse + rows + i));
        if (of_k) t *= dot((const T *)a.dout.row(b, i, h), v, a.D) + load_global<float>(a.delta + rows + i);
      }
      for (int u = 0; u < 64; ++u) {
        const int iu = __shfl(i, u);
        const float tu = __shfl(t, u);
        if (iu < 0) break;
        const T *r = of_k ? (const T *)a.q.row(b, iu, h) : (const T *)a.dout.row(b, iu, h);
#pragma unroll
        for (int x = 0; x < 4; ++x)
          if (x * 64 + lane < a.D) acc[x] = __builtin_fmaf(tu, to_float(r + x * 64 + lane), acc[x]);
      }
      nan = all_nan(acc);
    }
  }
  T *to = (T *)(of_k ? a.dk.row(b, j, kh) : a.dv.row(b, j, kh));
#pragma unroll
  for (int x = 0; x < 4; ++x)
    if (x * 64 + lane < a.D) {
      const float t[1] = {of_k ? acc[x] * a.scale : acc[x]};
      LaneVec<T, 1>::store(to + x * 64 + lane, LaneVec<T, 1>::pack(t));
    }
}

// ---- a lane's token of the side that stays in registers ----
// Operands of one token per lane: channels 16 s + 8 h ..; zeros past the head.
template <typename T, int DP> __device__ __forceinline__ void load_token(const T *p, int D, operand_t<T> (&f)[DP / 16]) {
  const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    const int d = 16 * s + 8 * h;
    operand_t<T> z = {};
    if (d < D) {
      if constexpr (sizeof(T) == 2) {
        z = load_global<operand_t<T>>(p + d);
      } else {
        const f32x4 x = load_global<f32x4>(p + d), y = load_global<f32x4>(p + d + 4);
        z = f32x8_t{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
      }
    }
    f[s] = z;
  }
}
// Waits for them here: a wait in the loop would be one for all copies on their way, too.
template <typename O, int N> __device__ __forceinline__ void settle(O (&f)[N]) {
#pragma unroll
  for (int x = 0; x < N; ++x) pin(f[x]);
}
// Channels of one token per lane from a transposed result, times `factor`, rounded once.
template <typename T, int DP> __device__ __forceinline__ void store_token(T *p, int D, const f32x16_t (&acc)[DP / 32], float factor) {
  const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int c = 0; c < DP / 32; ++c)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int d = 32 * c + row_of(r, h);
      if (d < D) {
        const float t[4] = {acc[c][r] * factor, acc[c][r + 1] * factor, acc[c][r + 2] * factor, acc[c][r + 3] * factor};
        using LV = LaneVec<T, 4>;
        LV::store(p + d, LV::pack(t));
      }
    }
}
// The same of 16-bit results, with REST what their rounding leaves instead, through a wavefront's own 64 DP bytes of shared memory, so
// that a row leaves in whole lines: row r goes to `to` + r row_bytes if r < last.  (Two results of 16 samples of 128 tokens, 8 heads
// of 128: the forward takes 9.0 us so, 10.0 by 8 bytes of a row at a time; the backward, with one result a kernel, is no faster.)
template <typename T, int DP, bool REST>
__device__ __forceinline__ void store_rows(char *place, const f32x16_t (&acc)[DP / 32], float factor, int D, char *to, int64_t row_bytes, int last) {
  static_assert(sizeof(T) == 2, "");
  using LV = LaneVec<T, 4>;
  constexpr int kChunks = DP / 8, kMask = (kChunks & -kChunks) - 1;  // (rows' chunks turned, so that they are not all in the same banks)
  const int lane = threadIdx.x & 63, h = lane >> 5, row = lane & 31;
#pragma unroll
  for (int c = 0; c < DP / 32; ++c)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const float t[4] = {acc[c][r] * factor, acc[c][r + 1] * factor, acc[c][r + 2] * factor, acc[c][r + 3] * factor};
      auto raw = LV::pack(t);
      if constexpr (REST) {
        float left[4];
        LV::unpack(raw, left);
#pragma unroll
        for (int e = 0; e < 4; ++e) left[e] = t[e] - left[e];
        raw = LV::pack(left);
      }
      *(decltype(raw) *)(place + (row * kChunks + ((4 * c + r / 4) ^ (row & kMask))) * 16 + h * 8) = raw;
    }
  asm volatile("" ::: "memory");
#pragma unroll
  for (int n = 0; n < kChunks / 2; ++n) {
    const int e = n * 64 + lane, r = e / kChunks, ch = e % kChunks;
    const u32x4 v = *(const u32x4 *)(place + (r * kChunks + (ch ^ (r & kMask))) * 16);
    if (r < last && ch * 8 < D) store_global<u32x4>(to + r * row_bytes + ch * 16, v);
  }
  asm volatile("" ::: "memory");
}
// Rows are written again, by other lanes: what they hold has to be there before.
__device__ __forceinline__ void rows_written() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
// The same for rows that any wavefront has written.
__device__ __forceinline__ void rows_of_all_written() {
  rows_written();
  __syncthreads();
}
// A token that sees nothing, or that nobody sees, gets zeros, whatever its tile held: its weights are 0, and 0 times NaN is NaN.
template <int N> __device__ __forceinline__ void clear_unless(bool kept, f32x16_t (&acc)[N]) {
#pragma unroll
  for (int x = 0; x < N; ++x)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[x][r] = kept ? acc[x][r] : 0.0f;
}
template <int N> __device__ __forceinline__ bool any_not_finite(const f32x16_t (&acc)[N]) {
  float t = 0.0f;
#pragma unroll
  for (int c = 0; c < N; ++c)
#pragma unroll
    for (int r = 0; r < 16; ++r) t = __builtin_fmaf(acc[c][r], 0.0f, t);
  return !(t == 0.0f);
}
__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32); }
__device__ __forceinline__ bool either_half(bool v) {
  const uint64_t m = __ballot(v);
  return ((m | m >> 32 | m << 32) >> (threadIdx.x & 63)) & 1;
}

// ---- forward ----
// The exponentials' reference is raised only when a score passes it by this much (in powers of two): the sums stay far inside a
// float's range, weights below 2^8 inside a float16's, and most tiles leave the accumulators alone.
constexpr float kRaise = 8.0f;

template <typename T, int DP> struct ForwardState {
  operand_t<T> q[DP / 16];
  f32x16_t o[DP / 32];
  float reference, subtract, sum;  // (sum: of the lane's half of the keys) in powers of two; subtract: the reference, or 0 while there is none
  Sight sight;
};

// 32 N keys against the wavefront's 32 queries: scores, then weights in their place, then their products with the values.  SUMS:
// float32 scores as sums of 16 channels' sums (half the error of adding channel to channel, for 16 additions a step, which a wavefront
// that waits for its keys has time for).
template <typename T, int DP, int N, bool SUMS, typename ST> __device__ __forceinline__ void forward_tile(ST &st, const LaneOffsets<T, DP> &at, const char *kt, char *vt, int j0, float c, bool fine) {
  const int h = (threadIdx.x & 63) >> 5;
  const Sight &g = st.sight;
  const int left = j0 - g.low;
  const bool inside = (left >= 0 && left + 32 * N <= g.count) || j0 + 32 * N <= g.sinks;
  if (!__all(inside) && !__any((left + 32 * N > 0 && left < g.count) || j0 < g.sinks)) return;
  f32x16_t s[N];
#pragma unroll
  for (int x = 0; x < DP / 16; ++x) {
    if (!at.has(x)) break;
    if constexpr (sizeof(T) == 4 && SUMS) {
      const f32x16_t t = Operand<T>::product(at.template of_rows<0>(kt, x), st.q[x], zeros16());
      s[0] = x ? s[0] + t : t;
    } else {
      s[0] = Operand<T>::product(at.template of_rows<0>(kt, x), st.q[x], x ? s[0] : zeros16());
    }
    if constexpr (N == 2) s[N - 1] = Operand<T>::product(at.template of_rows<32>(kt, x), st.q[x], x ? s[N - 1] : zeros16());
  }
  if (!__all(inside)) {
    int first = j0;
    pin(first);  // (so that the comparisons stay here)
#pragma unroll
    for (int f = 0; f < N; ++f)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (!g.sees(first + 32 * f + row_of(r, h))) s[f][r] = -INFINITY;
  }
  float most = s[0][0];
#pragma unroll
  for (int f = 0; f < N; ++f)
#pragma unroll
    for (int r = f ? 0 : 1; r < 16; ++r) most = fmaxf(most, s[f][r]);
  if (__any(most * c > st.reference + kRaise)) {
    most = fmaxf(most, other_half(most)) * c;
    const float reference = fmaxf(most, st.reference);
    const float factor = reference == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(st.reference - reference);
    st.reference = reference;
    st.subtract = reference == -INFINITY ? 0.0f : reference;
    st.sum *= factor;
#pragma unroll
    for (int x = 0; x < DP / 32; ++x)
#pragma unroll
      for (int r = 0; r < 16; ++r) st.o[x][r] *= factor;
  }
  auto part = [&](auto unit) {  // 16 keys
    constexpr int u = decltype(unit)::value;
    f32x16_t &p = s[u / 2];
#pragma unroll
    for (int r = 8 * (u % 2); r < 8 * (u % 2) + 8; ++r) {
      p[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[r], c, -st.subtract));
      st.sum += p[r];
    }
    const operand_t<T> w = operand_of<T>(p, u % 2);
#pragma unroll
    for (int x = 0; x < DP / 32; ++x) st.o[x] = Operand<T>::product(at.template of_columns<16 * u>(vt, x), w, st.o[x]);
    if constexpr (sizeof(T) == 2) {
      if (fine) {  // and what the weights' rounding left
#pragma unroll
        for (int r = 0; r < 8; ++r) p[8 * (u % 2) + r] -= (float)w[r];
        const operand_t<T> left = operand_of<T>(p, u % 2);
#pragma unroll
        for (int x = 0; x < DP / 32; ++x) st.o[x] = Operand<T>::product(at.template of_columns<16 * u>(vt, x), left, st.o[x]);
      }
    }
  };
  part(std::integral_constant<int, 0>());
  part(std::integral_constant<int, 1>());
  if constexpr (N == 2) {
    part(std::integral_constant<int, 2>());
    part(std::integral_constant<int, 3>());
  }
}

// Steps of a walk that one of `splits` workgroups takes: begin .. end - 1.
struct Stretch {
  Walk w;
  int begin, end;
  __device__ __forceinline__ int tile(int u) const { return u < w.sinks ? u : w.first + (u - w.sinks); }
  // Whether step u + by does not come `by` tiles behind step u.
  __device__ __forceinline__ bool jumps(int u, int by) const { return u < w.sinks && u + by >= w.sinks && w.first != w.sinks; }
};
// Of `steps` steps the n-th share begins at this one (the first ones are longer by one where they do not come out even).
__device__ __forceinline__ int share_begin(const Divisor &shares, int steps, int n) {
  const int each = div_by(steps, shares), more = steps - each * shares.d;
  return each * n + (n < more ? n : more);
}
__device__ __forceinline__ Stretch stretch_of(const Walk &w, int split, const Divisor &splits) {
  const int steps = w.sinks + (w.last >= w.first ? w.last - w.first + 1 : 0);
  return {w, share_begin(splits, steps, split), share_begin(splits, steps, split + 1)};
}
// Rows of the results of workgroups that share a row's keys: a split's rows behind each other, then the next split's.
__device__ __forceinline__ int64_t part_row(const WindowArgs &a, int split, int b, int h, int i) {
  return (((int64_t)split * a.B + b) * a.H + h) * a.L + i;
}

// A workgroup: 128 queries of one head, 32 a wavefront, against one of `splits` shares of the keys that they see.  128 queries share a
// tile's copy; 64 keys a tile are as many as leave room for four workgroups of heads of 64 in a CU's registers, whose waits hide
// each other.  float16 15600 tokens, 8 heads of 128, window 2400: 314 to 330 us a pass, 860 to 900 TFLOP/s (a library's product 1070); bfloat16 4 x
// 4096, 20 heads of 64: 810; with window 512, where a tenth of the pairs of its tiles is hidden, 675.  FINE: a.fine, as a
// kernel of its own (float16 heads of 64 have no registers left for both in one, and few queries are 3 % slower with both).
template <typename T, int DP, bool FINE>
__global__ __launch_bounds__(kBlock, sizeof(T) == 4 ? 2 : DP <= 64 && !FINE ? 4 : DP <= 128 ? 2 : 1) void window_forward_kernel(const WindowArgs a) {
  using G = Tile<T, DP>;
  __shared__ __attribute__((aligned(16))) char tiles[4 * G::kBytes];  // keys and values, two deep
  const int item = work_item(a);
  if (item >= a.items) return;
  // (the heads of a group are neighbours, then the tiles of queries, the last ones, which see most, first)
  const int of_group = div_by(item, a.by_group), rest = div_by(of_group, a.by_splits), g = item - of_group * a.group, split = of_group - rest * a.splits;
  const int bk = div_by(rest, a.by_tiles), tile = a.tiles - 1 - (rest - bk * a.tiles);
  const int b = div_by(bk, a.by_K), kh = bk - b * a.K, h = kh * a.group + g;
  const Sample s = sample_of(a, b);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), i = tile * kQueries + wave * 32 + (lane & 31);
  ForwardState<T, DP> st;
  st.sight = sight_of(a, s, i);
  st.reference = -INFINITY;
  st.subtract = 0.0f;
  st.sum = 0.0f;
#pragma unroll
  for (int x = 0; x < DP / 32; ++x) st.o[x] = zeros16();
  const int from = tile * kQueries > s.first ? tile * kQueries : s.first, to = (tile + 1) * kQueries < s.last ? (tile + 1) * kQueries : s.last;
  if (from < to) {
    const int ic = i < from ? from : i < to ? i : to - 1;
    load_token<T, DP>((const T *)a.q.row(b, ic, h), a.D, st.q);
    const Stretch w = stretch_of(walk_of(a, s, from + s.off, to - 1 + s.off, G::kRows), split, a.by_splits);
    TilePair<T, DP, G::kRows, kBlock> copy;
    copy.init(a.D, a.k.token_bytes, a.v.token_bytes, s.n - 1);
    LaneOffsets<T, DP> at;
    at.init(a.D);
    const char *kb = (const char *)a.k.row(b, 0, kh), *vb = (const char *)a.v.row(b, 0, kh);
    const unsigned lds = lds_address(tiles) + wave * 1024;
    auto issue = [&](int u, int buffer) {  // tile u, which is the next one; then the one behind it is
      copy.issue(lds + buffer * 2 * G::kBytes, G::kBytes);
      if (w.jumps(u, 1)) copy.go_to(kb, vb, w.tile(u + 1) * G::kRows);
      else copy.advance(1);
    };
    copy.go_to(kb, vb, w.tile(w.begin) * G::kRows);
    settle(st.q);
    int u = w.begin;
    if (u < w.end) issue(u, 0);
    auto turn = [&](auto buffer) {
      constexpr int B = decltype(buffer)::value;
      tiles_turn();
      if (u + 1 < w.end) issue(u + 1, 1 - B);
      forward_tile<T, DP, G::kRows / 32, false>(st, at, tiles + B * 2 * G::kBytes, tiles + B * 2 * G::kBytes + G::kBytes, w.tile(u) * G::kRows, a.scale_log2, FINE);
      ++u;
    };
    while (u < w.end) {
      turn(std::integral_constant<int, 0>());
      if (u >= w.end) break;
      turn(std::integral_constant<int, 1>());
    }
  }
  const WindowArgs &z = arguments_again();
  const float sum = st.sum + other_half(st.sum);
  const int i0 = tile * kQueries + wave * 32;
  const bool there = i < z.L, seeing = st.sight.count > 0 || st.sight.sinks > 0;
  clear_unless(seeing, st.o);
  if (z.splits > 1) {
    if (there) {
      const int64_t row = part_row(z, split, b, h, i);
      store_token<float, DP>(z.part_v + row * z.D, z.D, st.o, 1.0f);
      if (lane < 32) {
        store_global<float>(z.part_k + 2 * row, st.reference);
        store_global<float>(z.part_k + 2 * row + 1, sum);
      }
    }
    return;
  }
  const bool nothing = !(sum > 0.0f);  // (no key seen, or no score above -inf: those that see one are computed again)
  const float factor = nothing ? 0.0f : 1.0f / sum;
  const bool again = either_half(any_not_finite(st.o) || !(factor < INFINITY) || nothing) && seeing;
  if constexpr (sizeof(T) == 2) {
    char *place = tiles + wave * G::kBytes;
    __syncthreads();  // (the tiles have been read)
    if (i0 < z.L) {
      store_rows<T, DP, false>(place, st.o, factor, z.D, z.out.row(b, i0, h), z.out.token_bytes, z.L - i0);
      if (z.rest)
        store_rows<T, DP, true>(place, st.o, factor, z.D, (char *)((T *)z.rest + (((int64_t)b * z.L + i0) * z.H + h) * z.D), (int64_t)z.H * z.D * 2, z.L - i0);
    }
  } else if (there) {
    store_token<T, DP>((T *)z.out.row(b, i, h), z.D, st.o, factor);
  }
  if (z.lse && there && lane < 32) store_global<float>(z.lse + ((int64_t)b * z.H + h) * z.L + i, nothing ? INFINITY : st.reference + __builtin_amdgcn_logf(sum));
  uint64_t rows = __ballot(again && there) & 0xffffffffu;
  if (rows) rows_written();
  while (rows) {
    const int r = __builtin_ctzll(rows);
    rows &= rows - 1;
    row_again<T>(z, s, b, h, i0 + r);
  }
}

// ---- forward of few queries: the newest tokens of requests ----
// Rows (tokens times the heads of a group) fill one tile of 32, and the keys are what takes time: a workgroup is as many wavefronts
// as have room for two tiles of 32 keys and values each, every one walks keys of its own, and what they found is joined at the end.
// No barrier on the way: a wavefront waits for its own copies only.  64 requests of 32 heads over 8 of 128, 4100 keys: 184 us, 5.6 TB/s;
// one of 24 heads over 8, 517 keys: 8 us, the latency of its arguments, its tile and the join, and 4 of the second launch.  Where there are fewer heads than the device has room for,
// several workgroups share a head's keys (splits) and window_join_kernel joins them.
template <typename T, int DP> struct Few {
  static constexpr int kStage = 2 * 32 * DP * (int)sizeof(T);  // bytes of a tile of keys and one of values
  static constexpr int kWaves = few_waves(DP, sizeof(T));
  static constexpr int kPitch = DP + 4;                     // floats of a row while results are joined
  static_assert(32 * kPitch * 4 <= 2 * kStage, "a wavefront's results fit its tiles");
};
// Takes the next tile of a wavefront's own walk: COPIES copies of another one, if there is one, are issued by issue(), into the place of
// the one before.  Two tiles are on their way while the wavefront waits for the older one.  (That counts the newest copies: nothing
// else may be among them, so that these kernels must keep no register in scratch memory.)
template <int COPIES, typename F> __device__ __forceinline__ void next_copies(bool more, F &&issue) {
  static_assert(COPIES < 64, "what the counter holds");
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (reads of the tile that is now overwritten)
  if (more) {
    issue();
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(COPIES) : "memory");
  } else {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }
}

// Weight and result of a row that is joined of parts: (reference, sum).
__device__ __forceinline__ float part_weight(float reference, float most) { return most == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(reference - most); }

template <typename T, int DP, bool FINE> __global__ __launch_bounds__((64 * Few<T, DP>::kWaves), 1) void window_few_kernel(const WindowArgs a) {
  using W = Few<T, DP>;
  constexpr int kWaves = W::kWaves;
  __shared__ __attribute__((aligned(16))) char tiles[kWaves * 2 * W::kStage];
  __shared__ float references[kWaves][32], sums[kWaves][32];
  __shared__ int bad[32];
  const int item = work_item(a);
  if (item >= a.items) return;
  const int rest = div_by(item, a.by_splits), split = item - rest * a.splits, bk = div_by(rest, a.by_tiles), block = rest - bk * a.tiles;
  const int b = div_by(bk, a.by_K), kh = bk - b * a.K;
  const Sample s = sample_of(a, b);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int rows = a.L * a.group, row = block * 32 + (lane & 31), i = row < rows ? div_by(row, a.by_group) : a.L, h = kh * a.group + rest_by(row, a.by_group);
  ForwardState<T, DP> st;
  st.sight = sight_of(a, s, i);
  st.reference = -INFINITY;
  st.subtract = 0.0f;
  st.sum = 0.0f;
#pragma unroll
  for (int x = 0; x < DP / 32; ++x) st.o[x] = zeros16();
  int from = div_by(block * 32, a.by_group), to = div_by(block * 32 + 31, a.by_group) + 1;
  from = from > s.first ? from : s.first;
  to = to < s.last ? to : s.last;
  if (from < to) {
    const int ic = i < from ? from : i < to ? i : to - 1;
    load_token<T, DP>((const T *)a.q.row(b, ic, h), a.D, st.q);
    const Stretch w = stretch_of(walk_of(a, s, from + s.off, to - 1 + s.off, 32), split, a.by_splits);
    const char *kb = (const char *)a.k.row(b, 0, kh), *vb = (const char *)a.v.row(b, 0, kh);
    TilePair<T, DP, 32, 64> copy;
    copy.init(a.D, a.k.token_bytes, a.v.token_bytes, s.n - 1);
    LaneOffsets<T, DP> at;
    at.init(a.D);
    const unsigned lds = lds_address(tiles) + wave * 2 * W::kStage;
    settle(st.q);
    auto issue = [&](int u, int buffer) {
      copy.issue(lds + buffer * W::kStage, W::kStage / 2);
      if (w.jumps(u, kWaves)) copy.go_to(kb, vb, w.tile(u + kWaves) * 32);
      else copy.advance(kWaves);
    };
    copy.go_to(kb, vb, w.tile(w.begin + wave) * 32);
    int u = w.begin + wave, turn = 0;
    if (u < w.end) issue(u, 0);
    for (; u < w.end; u += kWaves) {
      char *tile = tiles + (wave * 2 + turn) * W::kStage;
      turn ^= 1;
      next_copies<2 * TileCopy<T, DP, 32, 64>::kCopies>(u + kWaves < w.end, [&] { issue(u + kWaves, turn); });
      forward_tile<T, DP, 1, true>(st, at, tile, tile + W::kStage / 2, w.tile(u) * 32, a.scale_log2, FINE);
    }
  }
  const WindowArgs &z = arguments_again();
  // join the wavefronts
  clear_unless(st.sight.count > 0 || st.sight.sinks > 0, st.o);
  st.sum += other_half(st.sum);
  if (lane < 32) {
    references[wave][lane] = st.reference;
    sums[wave][lane] = st.sum;
    if (wave == 0) bad[lane] = 0;
  }
  __syncthreads();
  float most = -INFINITY, sum = 0.0f;
#pragma unroll
  for (int n = 0; n < kWaves; ++n) most = fmaxf(most, references[n][lane & 31]);
#pragma unroll
  for (int n = 0; n < kWaves; ++n) sum += sums[n][lane & 31] * part_weight(references[n][lane & 31], most);
  const float weight = part_weight(st.reference, most);
  float *mine = (float *)(tiles + wave * 2 * W::kStage);
  const int half = lane >> 5;
#pragma unroll
  for (int x = 0; x < DP / 32; ++x)
#pragma unroll
    for (int r = 0; r < 16; r += 4)
      *(f32x4 *)(mine + (lane & 31) * W::kPitch + 32 * x + row_of(r, half)) =
          f32x4{st.o[x][r] * weight, st.o[x][r + 1] * weight, st.o[x][r + 2] * weight, st.o[x][r + 3] * weight};
  __syncthreads();  // (also: all have read references and sums)
  if (wave == 0 && lane < 32) {
    references[0][lane] = most;
    sums[0][lane] = sum;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < 32 * DP / 4; e += 64 * kWaves) {
    const int r = e / (DP / 4), d = e % (DP / 4) * 4, rr = block * 32 + r;
    if (rr >= rows || d >= z.D) continue;
    f32x4 v = *(const f32x4 *)((const float *)tiles + r * W::kPitch + d);
#pragma unroll
    for (int n = 1; n < kWaves; ++n) v += *(const f32x4 *)((const float *)(tiles + n * 2 * W::kStage) + r * W::kPitch + d);
    if (z.splits > 1) {
      store_global<f32x4>(z.part_v + part_row(z, split, b, kh * z.group + rest_by(rr, z.by_group), div_by(rr, z.by_group)) * z.D + d, v);
      continue;
    }
    const float total = sums[0][r], factor = total > 0.0f ? 1.0f / total : 0.0f;
    const float t[4] = {v[0] * factor, v[1] * factor, v[2] * factor, v[3] * factor};
    if (!(v[0] * 0.0f + v[1] * 0.0f + v[2] * 0.0f + v[3] * 0.0f + factor * 0.0f == 0.0f) || !(total > 0.0f)) bad[r] = 1;
    store_out<T, 4>(z, b, kh * z.group + rest_by(rr, z.by_group), div_by(rr, z.by_group), d, t);
  }
  if (z.splits > 1) {
    const int rr = block * 32 + (int)threadIdx.x;
    if (threadIdx.x < 32 && rr < rows) {
      float *p = z.part_k + 2 * part_row(z, split, b, kh * z.group + rest_by(rr, z.by_group), div_by(rr, z.by_group));
      store_global<float>(p, references[0][threadIdx.x]);
      store_global<float>(p + 1, sums[0][threadIdx.x]);
    }
    return;
  }
  __syncthreads();
  const bool ours = lane < 32 && row < rows;
  if (z.lse && wave == 0 && ours)
    store_global<float>(z.lse + ((int64_t)b * z.H + h) * z.L + i, sums[0][lane] > 0.0f ? references[0][lane] + __builtin_amdgcn_logf(sums[0][lane]) : INFINITY);
  uint64_t again = __ballot(ours && bad[lane & 31] && (st.sight.count > 0 || st.sight.sinks > 0));  // (the same in all wavefronts)
  if (again) rows_of_all_written();
  while (again) {
    const int r = __builtin_ctzll(again);
    again &= again - 1;
    if (r % kWaves == wave) row_again<T>(z, s, b, __builtin_amdgcn_readlane(h, r), __builtin_amdgcn_readlane(i, r));
  }
}

// ---- joining ----
// Rows of results that several workgroups left parts of.  A thread has four channels of a row and about four of its parts (a few
// reads on their way at once); where there are more threads than one for that, they add up in shared memory, in their order.  43
// parts of the sinks' gradients, 3 samples of 2 heads of 40 channels in float32: 20 us by one thread, 7 by eleven.
struct Joining {
  int joiners, rows_here;  // threads that share the parts; rows of a workgroup
  Divisor lanes, quads;    // threads of a row, of a part of it
  Joining(int D, int parts) {
    const int room = kBlock / (D / 4), wanted = (parts + 3) / 4, n = wanted < room ? wanted : room;
    joiners = n < 1 ? 1 : n > 16 ? 16 : n;
    quads = make_divisor(D / 4, 0);
    lanes = make_divisor(quads.d * joiners, 0);
    rows_here = kBlock / lanes.d;
  }
  int64_t blocks(int64_t rows) const { return (rows + rows_here - 1) / rows_here; }
};
struct Joiner {
  int joiners, rows_here, row, part, d, quads;  // the thread's row of the workgroup's, its first part and first channel
  __device__ __forceinline__ explicit Joiner(const Joining &j) {
    joiners = j.joiners;
    rows_here = j.rows_here;
    quads = j.quads.d;
    row = div_by(threadIdx.x, j.lanes);
    const int left = threadIdx.x - row * j.lanes.d;
    part = div_by(left, j.quads);
    d = (left - part * quads) * 4;
  }
};
template <typename V, typename F> __device__ __forceinline__ V joined(const Joiner &at, V v, V *place, F &&f) {
  if (at.joiners == 1) return v;
  __syncthreads();
  place[threadIdx.x] = v;
  __syncthreads();
  if (at.row >= at.rows_here) return v;  // (left over: no row, and no parts in reach)
  const V *first = place + (threadIdx.x - at.part * at.quads);
  v = first[0];
  for (int n = 1; n < at.joiners; ++n) v = f(v, first[n * at.quads]);
  return v;
}

// (Eight workgroups a CU, which leaves 64 registers and 80 scalar ones: with a few more of either 30540 rows of 64 channels, three parts
// each, take 8.4 us for 7.0.)
template <typename T> __global__ __launch_bounds__(kBlock, 8) void window_join_kernel(const WindowArgs a, const Joining joining) {
  __shared__ int bad[kBlock], any_bad;
  __shared__ f32x4 place[kBlock];
  const Joiner at(joining);
  const int r = at.row, d = at.d, rows_here = at.rows_here;
  const int64_t rows = (int64_t)a.B * a.H * a.L;
  const int id = (int)blockIdx.x * rows_here + r;  // (fewer than 2^31: 128 of each of 2^23 workgroups)
  const bool there = r < rows_here && id < rows;
  bad[threadIdx.x] = 0;
  if (threadIdx.x == 0) any_bad = 0;
  const auto add = [](auto x, auto y) { return x + y; };
  float most = -INFINITY, sum = 0.0f;
  f32x4 o = {};
  if (there) {
#pragma unroll 4
    for (int n = at.part; n < a.splits; n += at.joiners) most = fmaxf(most, load_global<float>(a.part_k + 2 * (id + n * rows)));
  }
  most = joined(at, most, (float *)place, [](float x, float y) { return fmaxf(x, y); });
  if (there) {
#pragma unroll 4
    for (int n = at.part; n < a.splits; n += at.joiners) {
      const f32x2 part = load_global<f32x2>(a.part_k + 2 * (id + n * rows));
      const float w = part_weight(part.x, most);
      const f32x4 v = load_global<f32x4>(a.part_v + (id + n * rows) * a.D + d);
      sum = __builtin_fmaf(w, part.y, sum);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(w, v[e], o[e]);
    }
  }
  sum = joined(at, sum, (float *)place, add);
  o = joined(at, o, place, add);
  if (at.joiners == 1) __syncthreads();  // (bad is cleared)
  if (there && at.part == 0) {
    const float factor = sum > 0.0f ? 1.0f / sum : 0.0f;
    const float t[4] = {o[0] * factor, o[1] * factor, o[2] * factor, o[3] * factor};
    const int bh = div_by(id, a.by_L), i = id - bh * a.L, b = div_by(bh, a.by_H), h = bh - b * a.H;
    store_out<T, 4>(a, b, h, i, d, t);
    if (a.lse && d == 0) store_global<float>(a.lse + id, sum > 0.0f ? most + __builtin_amdgcn_logf(sum) : INFINITY);
    if (!(t[0] * 0.0f + t[1] * 0.0f + t[2] * 0.0f + t[3] * 0.0f == 0.0f) || !(sum > 0.0f)) bad[r] = any_bad = 1;
  }
  __syncthreads();
  if (!any_bad) return;
  rows_of_all_written();
  for (int n = threadIdx.x >> 6; n < rows_here; n += 4) {
    if (!bad[n]) continue;
    const WindowArgs &z = arguments_again();
    const int row = (int)blockIdx.x * rows_here + n;
    const int bh = div_by(row, z.by_L), i = row - bh * z.L, b = div_by(bh, z.by_H), h = bh - b * z.H;
    const Sample s = sample_of(z, b);
    const Sight g = sight_of(z, s, i);
    if (g.count > 0 || g.sinks > 0) row_again<T>(z, s, b, h, i);
  }
}

// ---- backward: dq ----
// -delta and the largest |do| of a row go to the workspace for the other kernel.
// float16 holds 2^-24 to 65504: weights and dS are kept in its middle by powers of two, weights as 2^12 P, dS relative to the
// largest |do| (of a row, or of the rows that a workgroup visits), whatever scale a loss has been given.
constexpr float kWeightBits = 12.0f, kGradBits = 5.0f;
template <typename T> __device__ __forceinline__ float gradient_unit(float most) {  // a power of two near 1 / most
  if constexpr (!__is_same(T, f16_t)) return 1.0f;
  else return most > 0.0f && most < INFINITY ? __builtin_amdgcn_ldexpf(1.0f, -__builtin_amdgcn_frexp_expf(most)) : 1.0f;
}

// A workgroup: 128 queries of one head against a share of the keys that they see, like the forward, with q and do in registers and
// three products a pair.  bfloat16, 4 x 4112 tokens, 20 heads of 64, window 512: 163 to 175 us, 121 GFLOP of the formula's at 0.7 PFLOP/s;
// without its copies 5 % less, without the exponentials a tenth, without the products a fifth: no one unit bounds it.
template <typename T, int DP> __global__ __launch_bounds__(kBlock, DP <= (sizeof(T) == 2 ? 128 : 96) ? 2 : 1) void window_dq_kernel(const WindowArgs a) {
  using G = Tile<T, DP>;
  __shared__ __attribute__((aligned(16))) char tiles[4 * G::kBytes];  // keys and values, two deep
  const int item = work_item(a);
  if (item >= a.items) return;
  const int of_group = div_by(item, a.by_group), rest = div_by(of_group, a.by_splits), g = item - of_group * a.group, split = of_group - rest * a.splits;
  const int bk = div_by(rest, a.by_tiles), tile = a.tiles - 1 - (rest - bk * a.tiles);
  const int b = div_by(bk, a.by_K), kh = bk - b * a.K, h = kh * a.group + g;
  const Sample s = sample_of(a, b);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), half = lane >> 5, i = tile * kQueries + wave * 32 + (lane & 31);
  const Sight sight = sight_of(a, s, i);
  const int64_t row = ((int64_t)b * a.H + h) * a.L + i;
  f32x16_t acc[DP / 32];
#pragma unroll
  for (int x = 0; x < DP / 32; ++x) acc[x] = zeros16();
  float lse = INFINITY, delta = 0.0f, unit = 1.0f;
  const int from = tile * kQueries > s.first ? tile * kQueries : s.first, to = (tile + 1) * kQueries < s.last ? (tile + 1) * kQueries : s.last;
  if (from < to) {
    const int ic = i < from ? from : i < to ? i : to - 1;
    operand_t<T> q[DP / 16], dout[DP / 16];
    load_token<T, DP>((const T *)a.dout.row(b, ic, h), a.D, dout);
    {
      load_token<T, DP>((const T *)a.out.row(b, ic, h), a.D, q);  // (o, for delta; q's place)
      float most = 0.0f;
#pragma unroll
      for (int x = 0; x < DP / 16; ++x)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          delta = __builtin_fmaf((float)dout[x][e], (float)q[x][e], delta);
          most = fmaxf(most, fabsf((float)dout[x][e]));
        }
      if constexpr (sizeof(T) == 2) {
        if (a.rest) {
          load_token<T, DP>((const T *)a.rest + (((int64_t)b * a.L + ic) * a.H + h) * a.D, a.D, q);
#pragma unroll
          for (int x = 0; x < DP / 16; ++x)
#pragma unroll
            for (int e = 0; e < 8; ++e) delta = __builtin_fmaf((float)dout[x][e], (float)q[x][e], delta);
        }
      }
      delta += other_half(delta);
      most = fmaxf(most, other_half(most));
      unit = gradient_unit<T>(most);
      if (split == 0 && i >= from && i < to && lane < 32) {
        store_global<float>(a.delta + row, -delta);
        if constexpr (__is_same(T, f16_t)) store_global<float>(a.largest + row, most);
      }
    }
    load_token<T, DP>((const T *)a.q.row(b, ic, h), a.D, q);
    if (i >= from && i < to) lse = load_global<float>(a.lse + row);
    const Stretch w = stretch_of(walk_of(a, s, from + s.off, to - 1 + s.off, G::kRows), split, a.by_splits);
    TilePair<T, DP, G::kRows, kBlock> copy;
    copy.init(a.D, a.k.token_bytes, a.v.token_bytes, s.n - 1);
    LaneOffsets<T, DP> at;
    at.init(a.D);
    const char *kb = (const char *)a.k.row(b, 0, kh), *vb = (const char *)a.v.row(b, 0, kh);
    const unsigned lds = lds_address(tiles) + wave * 1024;
    // P 2^bits (dP - delta) unit: the product starts from -delta
    const float bits = __is_same(T, f16_t) ? kGradBits : 0.0f;
    float lift = bits - lse;
    if constexpr (__is_same(T, f16_t)) lift += (float)__builtin_amdgcn_frexp_expf(unit) - 1.0f;  // (unit is 2^(its exponent - 1))
    f32x16_t start;
#pragma unroll
    for (int r = 0; r < 16; ++r) start[r] = -delta;
    settle(q);
    settle(dout);
    pin(lift);
    auto issue = [&](int u, int buffer) {  // tile u, which is the next one; then the one behind it is
      copy.issue(lds + buffer * 2 * G::kBytes, G::kBytes);
      if (w.jumps(u, 1)) copy.go_to(kb, vb, w.tile(u + 1) * G::kRows);
      else copy.advance(1);
    };
    copy.go_to(kb, vb, w.tile(w.begin) * G::kRows);
    int u = w.begin;
    if (u < w.end) issue(u, 0);
    auto turn = [&](auto buffer) {
      constexpr int B = decltype(buffer)::value;
      tiles_turn();
      if (u + 1 < w.end) issue(u + 1, 1 - B);
      const int place0 = w.tile(u) * G::kRows;
      char *kt = tiles + B * 2 * G::kBytes, *vt = kt + G::kBytes;
      auto part = [&](auto first) {
        constexpr int f = decltype(first)::value;
        const int j0 = place0 + f, left = j0 - sight.low;
        const bool inside = (left >= 0 && left + 32 <= sight.count) || j0 + 32 <= sight.sinks;
        const bool whole = __all(inside);
        if (!whole && !__any((left + 32 > 0 && left < sight.count) || j0 < sight.sinks)) return;
        f32x16_t p, dp;
#pragma unroll
        for (int x = 0; x < DP / 16; ++x) {
          if (!at.has(x)) break;
          p = Operand<T>::product(at.template of_rows<f>(kt, x), q[x], x ? p : zeros16());
          dp = Operand<T>::product(at.template of_rows<f>(vt, x), dout[x], x ? dp : start);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) p[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[r], a.scale_log2, lift)) * dp[r];
        if (!whole) {
          int from_here = j0;
          pin(from_here);  // (so that the comparisons stay here)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (!sight.sees(from_here + row_of(r, half))) p[r] = 0.0f;
        }
        const operand_t<T> ds0 = operand_of<T>(p, 0), ds1 = operand_of<T>(p, 1);
#pragma unroll
        for (int x = 0; x < DP / 32; ++x) acc[x] = Operand<T>::product(at.template of_columns<f>(kt, x), ds0, acc[x]);
#pragma unroll
        for (int x = 0; x < DP / 32; ++x) acc[x] = Operand<T>::product(at.template of_columns<f + 16>(kt, x), ds1, acc[x]);
      };
      part(std::integral_constant<int, 0>());
      if constexpr (G::kRows == 64) part(std::integral_constant<int, 32>());
      ++u;
    };
    while (u < w.end) {
      turn(std::integral_constant<int, 0>());
      if (u >= w.end) break;
      turn(std::integral_constant<int, 1>());
    }
  }
  const WindowArgs &z = arguments_again();
  const bool there = i < z.L, seeing = sight.count > 0 || sight.sinks > 0;
  clear_unless(seeing, acc);
  const bool again = either_half(any_not_finite(acc)) && seeing && there;
  if (there) {
    const float factor = seeing ? z.scale * (__is_same(T, f16_t) ? 1.0f / 32.0f / unit : 1.0f) : 0.0f;
    if (z.splits > 1) {
      store_token<float, DP>(z.part_q + part_row(z, split, b, h, i) * z.D, z.D, acc, factor);
      return;
    }
    store_token<T, DP>((T *)z.dq.row(b, i, h), z.D, acc, factor);
  }
  uint64_t rows = __ballot(again) & 0xffffffffu;
  if (rows) rows_written();
  while (rows) {
    const int r = __builtin_ctzll(rows);
    rows &= rows - 1;
    dq_again<T>(z, s, b, h, tile * kQueries + wave * 32 + r, __shfl(lse, r), __shfl(delta, r));
  }
}
static_assert(kGradBits == 5.0f, "the factors of 1 / 32 undo it");

// dq of rows whose keys several workgroups shared.
template <typename T> __global__ __launch_bounds__(kBlock, 8) void window_dq_sum_kernel(const WindowArgs a, const Joining joining) {
  __shared__ int bad[kBlock], any_bad;
  __shared__ f32x4 place[kBlock];
  const Joiner at(joining);
  const int r = at.row, rows_here = at.rows_here;
  const int64_t rows = (int64_t)a.B * a.H * a.L;
  const int id = (int)blockIdx.x * rows_here + r;  // (fewer than 2^31: 128 of each of 2^23 workgroups)
  const bool there = r < rows_here && id < rows;
  bad[threadIdx.x] = 0;
  if (threadIdx.x == 0) any_bad = 0;
  f32x4 q = {};
  if (there) {
#pragma unroll 4
    for (int n = at.part; n < a.splits; n += at.joiners) q += load_global<f32x4>(a.part_q + (id + n * rows) * a.D + at.d);
  }
  q = joined(at, q, place, [](f32x4 x, f32x4 y) { return x + y; });
  if (at.joiners == 1) __syncthreads();  // (bad is cleared)
  if (there && at.part == 0) {
    const float t[4] = {q[0], q[1], q[2], q[3]};
    using LV = LaneVec<T, 4>;
    const int bh = div_by(id, a.by_L), i = id - bh * a.L, b = div_by(bh, a.by_H), h = bh - b * a.H;
    LV::store((T *)a.dq.row(b, i, h) + at.d, LV::pack(t));
    if (!(q[0] * 0.0f + q[1] * 0.0f + q[2] * 0.0f + q[3] * 0.0f == 0.0f)) bad[r] = any_bad = 1;
  }
  __syncthreads();
  if (!any_bad) return;
  rows_of_all_written();
  for (int n = threadIdx.x >> 6; n < rows_here; n += 4) {
    if (!bad[n]) continue;
    const WindowArgs &z = arguments_again();
    const int row = (int)blockIdx.x * rows_here + n;
    const int bh = div_by(row, z.by_L), i = row - bh * z.L, b = div_by(bh, z.by_H), h = bh - b * z.H;
    const Sample s = sample_of(z, b);
    const Sight g = sight_of(z, s, i);
    if (g.count > 0 || g.sinks > 0) dq_again<T>(z, s, b, h, i, load_global<float>(z.lse + row), -load_global<float>(z.delta + row));
  }
}

// ---- backward: dk and dv ----
// Ends a phase of a kernel that reads its operands from shared memory a phase ahead of the products that take them: nothing is
// moved across (the compiler would read each right in front of its product and wait).
template <bool AHEAD> __device__ __forceinline__ void phase_end() {
  if constexpr (AHEAD) __builtin_amdgcn_sched_barrier(0);
}

// 32 keys of a wavefront, one a lane.  PARTS: 1 dv, 2 dk, 3 both (heads of more than 128 channels, in float32 96, do not fit the registers at once).
template <typename T, int DP, int PARTS> struct KeySide {
  static constexpr bool kDv = PARTS & 1, kDk = PARTS & 2;
  static constexpr bool kAhead = DP <= (sizeof(T) == 2 ? 128 : 64);
  operand_t<T> k[DP / 16], v[kDk ? DP / 16 : 1];
  f32x16_t dk[kDk ? DP / 32 : 1], dv[kDv ? DP / 32 : 1];
  Seen seen;
  float c, lowering;  // scale; float16: 2^(kGradBits - kWeightBits) times the unit of the gradients

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int x = 0; x < DP / 32; ++x) {
      if constexpr (kDk) dk[x] = zeros16();
      if constexpr (kDv) dv[x] = zeros16();
    }
  }
  __device__ __forceinline__ void clear_unseen() {
    if constexpr (kDk) clear_unless(seen.count > 0, dk);
    if constexpr (kDv) clear_unless(seen.count > 0, dv);
  }
  __device__ __forceinline__ void load(const WindowArgs &a, int b, int j, int kh) {
    load_token<T, DP>((const T *)a.k.row(b, j, kh), a.D, k);
    if constexpr (kDk) load_token<T, DP>((const T *)a.v.row(b, j, kh), a.D, v);
  }
  __device__ __forceinline__ void settle_operands() {
    settle(k);
    if constexpr (kDk) settle(v);
  }
  // ROWS queries, the first at place `place`; their lse and -delta lie beside the tiles.
  template <int ROWS> __device__ __forceinline__ void tile(const LaneOffsets<T, DP> &at, char *qt, char *gt, const float *lses, const float *deltas, int place) {
    const int half = (threadIdx.x & 63) >> 5;
    if (!__any(place + ROWS > seen.from && place < seen.from + seen.count)) return;
    operand_t<T> qr[DP / 16], gr[kDk ? DP / 16 : 1];
    f32x16_t dp;
    auto read_rows = [&](auto first_row) {
      constexpr int f = decltype(first_row)::value;
#pragma unroll
      for (int x = 0; x < DP / 16; ++x) qr[x] = at.template of_rows<f>(qt, x);
      if constexpr (kDk) {
#pragma unroll
        for (int r = 0; r < 16; r += 4) {  // (the product starts from -delta)
          const f32x4 d4 = *(const f32x4 *)&deltas[f + row_of(r, half)];
#pragma unroll
          for (int e = 0; e < 4; ++e) dp[r + e] = d4[e];
        }
#pragma unroll
        for (int x = 0; x < DP / 16; ++x) gr[x] = at.template of_rows<f>(gt, x);
      }
    };
    auto part = [&](auto first_row, auto is_last) {
      constexpr int f = decltype(first_row)::value;
      f32x16_t p, lse;
#pragma unroll
      for (int x = 0; x < DP / 16; ++x) {
        if (!at.has(x)) break;
        p = Operand<T>::product(qr[x], k[x], x ? p : zeros16());
      }
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const f32x4 l4 = *(const f32x4 *)&lses[f + row_of(r, half)];
#pragma unroll
        for (int e = 0; e < 4; ++e) lse[r + e] = l4[e];
      }
      operand_t<T> gc[kDv ? DP / 32 : 1][2], qc[kDk ? DP / 32 : 1][2];
      if constexpr (kDv) {
#pragma unroll
        for (int x = 0; x < DP / 32; ++x) gc[x][0] = at.template of_columns<f>(gt, x), gc[x][1] = at.template of_columns<f + 16>(gt, x);
      }
      phase_end<kAhead>();
      if constexpr (kDk) {
#pragma unroll
        for (int x = 0; x < DP / 16; ++x) {
          if (!at.has(x)) break;
          dp = Operand<T>::product(gr[x], v[x], dp);
        }
#pragma unroll
        for (int x = 0; x < DP / 32; ++x) qc[x][0] = at.template of_columns<f>(qt, x), qc[x][1] = at.template of_columns<f + 16>(qt, x);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) p[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[r], c, __is_same(T, f16_t) ? kWeightBits - lse[r] : -lse[r]));
      if (!__all(place + f >= seen.from && place + f + 32 <= seen.from + seen.count)) {
        int left = place + f - seen.from;
        pin(left);  // (so that the comparisons stay here)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const bool hidden = (unsigned)(left + row_of(r, half)) >= (unsigned)seen.count;
          if (hidden) p[r] = 0.0f;
          if constexpr (kDk) {
            if (hidden) dp[r] = 0.0f;  // (which may be infinite)
          }
        }
      }
      phase_end<kAhead>();
      if constexpr (kDv) {
        const operand_t<T> w[2] = {operand_of<T>(p, 0), operand_of<T>(p, 1)};
#pragma unroll
        for (int x = 0; x < DP / 32; ++x)
#pragma unroll
          for (int u = 0; u < 2; ++u) dv[x] = Operand<T>::product(gc[x][u], w[u], dv[x]);
      }
      if constexpr (kDk) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          if constexpr (__is_same(T, f16_t)) p[r] *= lowering;
          p[r] *= dp[r];
        }
      }
      if constexpr (!decltype(is_last)::value) read_rows(std::integral_constant<int, f + 32>());
      phase_end<kAhead>();
      if constexpr (kDk) {
        const operand_t<T> w[2] = {operand_of<T>(p, 0), operand_of<T>(p, 1)};
#pragma unroll
        for (int x = 0; x < DP / 32; ++x)
#pragma unroll
          for (int u = 0; u < 2; ++u) dk[x] = Operand<T>::product(qc[x][u], w[u], dk[x]);
      }
    };
    read_rows(std::integral_constant<int, 0>());
    if constexpr (ROWS == 64) {
      part(std::integral_constant<int, 0>(), std::false_type());
      part(std::integral_constant<int, 32>(), std::true_type());
    } else {
      part(std::integral_constant<int, 0>(), std::true_type());
    }
  }
  static __device__ __forceinline__ float v_factor() { return __is_same(T, f16_t) ? 1.0f / 4096.0f : 1.0f; }
  static __device__ __forceinline__ float k_factor(const WindowArgs &a, float unit) { return a.scale * (__is_same(T, f16_t) ? 1.0f / 32.0f / unit : 1.0f); }
};
static_assert(kWeightBits == 12.0f, "the factors of 1 / 4096 and 1 / 128 undo it");

// The queries that see any of the keys j0 .. top - 1 (of the window, or as sinks): from .. to.
struct Queries {
  int from, to;
};
__device__ __forceinline__ Queries queries_of(const WindowArgs &a, const Sample &s, int j0, int top, bool sinks) {
  if (j0 >= top || s.first >= s.last) return {0, -1};
  const int least = s.first + s.off, most = s.last - 1 + s.off;
  const int lo = sinks ? (a.causal ? j0 : 0) : j0 - a.right, hi = sinks ? s.n - 1 : top - 1 + a.left;
  return {(lo > least ? lo : least) - s.off, (hi < most ? hi : most) - s.off};
}
// A step of a walk over queries: a head of the group, a tile.
struct Step {
  int g, t;
  __device__ __forceinline__ void advance(int by, int tiles) {
    t += by;
    while (t >= tiles) {
      t -= tiles;
      ++g;
    }
  }
};
// Where workgroups that share keys leave their sums of rows: first the sinks', 32 keys at a time, then those of tiles.
__device__ __forceinline__ int64_t sink_slot(const WindowArgs &a, int bk, int set, int part) { return (((int64_t)bk * a.sink_sets + set) * a.sink_parts + part) * 32; }
__device__ __forceinline__ int64_t tile_slot(const WindowArgs &a, int bk, int tile, int share) {
  return (int64_t)a.B * a.K * a.sink_sets * a.sink_parts * 32 + (((int64_t)bk * a.tiles + tile) * a.shares + share) * kQueries;
}

// A workgroup: 128 keys of one head, 32 a wavefront, against a share of the queries whose windows have any of them, of all heads of
// the group.  Where several share a tile's queries, each leaves float32 sums, which window_sum_kernel adds in their order.  Sinks,
// which all queries see, are left to window_sink_kernel.  k, v and both sums of 32 keys stay in registers, which leaves two wavefronts
// a SIMD for heads of 64 (three would have registers in scratch memory: 321 us for 254) and one beyond, and operands are read a phase
// ahead of their products instead.  bfloat16, 4 x 4112 tokens, 20 heads of 64, window 512: 197 to 212 us, 0.8 PFLOP/s; 2 x 4096, 24 over 8
// of 128, causal, window 1024: 238 to 258.
template <typename T, int DP, int PARTS>
__global__ __launch_bounds__(kBlock, (DP <= 64 && sizeof(T) == 2) || (sizeof(T) == 4 && PARTS == 1) ? 2 : 1) void window_dkv_kernel(const WindowArgs a) {
  using G = Tile<T, DP>;
  using KS = KeySide<T, DP, PARTS>;
  __shared__ __attribute__((aligned(16))) char tiles[4 * G::kBytes];  // queries and gradients, two deep
  __shared__ __attribute__((aligned(16))) float lses[2 * 64], deltas[2 * 64];
  __shared__ float reduce[4];
  const int item = work_item(a);
  if (item >= a.items) return;
  const int rest = div_by(item, a.by_shares), share = item - rest * a.shares, bk = div_by(rest, a.by_tiles), tile = rest - bk * a.tiles;
  const int b = div_by(bk, a.by_K), kh = bk - b * a.K;
  const Sample s = sample_of(a, b);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), j = tile * kQueries + wave * 32 + (lane & 31);
  const bool ours = j >= a.sinks && j < a.S;
  KS key;
  key.clear();
  key.seen = ours ? seen_of(a, s, j) : Seen{0, 0};
  key.c = a.scale_log2;
  float unit = 1.0f;
  const int j0 = tile * kQueries > a.sinks ? tile * kQueries : a.sinks, top = (tile + 1) * kQueries < s.n ? (tile + 1) * kQueries : s.n;
  const Queries range = queries_of(a, s, j0, top, false);
  if (range.from <= range.to) {
    const int first = range.from / G::kRows, tiles_of = range.to / G::kRows - first + 1, steps = tiles_of * a.group, to = range.to;
    const int begin = share_begin(a.by_shares, steps, share), end = share_begin(a.by_shares, steps, share + 1);
    if constexpr (__is_same(T, f16_t)) {
      float most = 0.0f;
      for (int st = begin + wave; st < end; st += 4) {
        const int64_t rows = ((int64_t)b * a.H + kh * a.group + st / tiles_of) * a.L;
        const int i = (first + st % tiles_of) * G::kRows + lane;
        if (i >= range.from && i <= to) most = fmaxf(most, load_global<float>(a.largest + rows + i));
      }
      most = wave_max(most);
      if (lane == 0) reduce[wave] = most;
      __syncthreads();
      unit = gradient_unit<T>(fmaxf(fmaxf(reduce[0], reduce[1]), fmaxf(reduce[2], reduce[3])));
    }
    key.lowering = unit * (1.0f / 128.0f);
    key.load(a, b, j < s.n ? j : s.n - 1, kh);
    TilePair<T, DP, G::kRows, kBlock> copy;
    copy.init(a.D, a.q.token_bytes, a.dout.token_bytes, to);
    LaneOffsets<T, DP> at;
    at.init(a.D);
    const unsigned lds = lds_address(tiles) + wave * 1024, lds_lse = lds_address(lses), lds_delta = lds_address(deltas);
    key.settle_operands();
    const float *at_row = nullptr;  // lse for the first wavefront, -delta for the second
    auto go_to = [&](Step w) {
      const int h = kh * a.group + w.g, i0 = (first + w.t) * G::kRows;
      copy.go_to((const char *)a.q.row(b, 0, h), (const char *)a.dout.row(b, 0, h), i0);
      at_row = uniform((wave ? a.delta : a.lse) + ((int64_t)b * a.H + h) * a.L + i0);
    };
    const unsigned lds_row = (wave ? lds_delta : lds_lse);
    int left_over = end - begin;
    Step step = {begin / tiles_of, begin % tiles_of}, next = step;
    auto issue = [&](int buffer) {  // tile `next`; then the one behind it is next
      copy.issue(lds + buffer * 2 * G::kBytes, G::kBytes);
      if (wave < (KS::kDk ? 2 : 1)) {
        const int r = to - copy.first;
        copy_to_lds<4>((const char *)at_row, (unsigned)(lane < r ? lane : r) * 4, lds_row + buffer * 256);
      }
      next.advance(1, tiles_of);
      if (next.t == 0) {
        go_to(next.g < a.group ? next : step);
      } else {
        copy.advance(1);
        at_row += G::kRows;
      }
    };
    go_to(step);
    if (left_over > 0) issue(0);
    auto turn = [&](auto buffer) {
      constexpr int B = decltype(buffer)::value;
      tiles_turn();
      const Step now = step;
      step = next;
      if (--left_over > 0) issue(1 - B);
      char *qt = tiles + B * 2 * G::kBytes;
      key.template tile<G::kRows>(at, qt, qt + G::kBytes, lses + B * 64, deltas + B * 64, (first + now.t) * G::kRows + s.off);
    };
    while (left_over > 0) {
      turn(std::integral_constant<int, 0>());
      if (left_over <= 0) break;
      turn(std::integral_constant<int, 1>());
    }
  }
  const WindowArgs &z = arguments_again();
  key.clear_unseen();
  if (z.shares > 1) {
    const int64_t slot = tile_slot(z, bk, tile, share) + wave * 32 + (lane & 31);
    if constexpr (KS::kDk) store_token<float, DP>(z.part_k + slot * z.D, z.D, key.dk, KS::k_factor(z, unit));
    if constexpr (KS::kDv) store_token<float, DP>(z.part_v + slot * z.D, z.D, key.dv, KS::v_factor());
    return;
  }
  if (ours) {
    if constexpr (KS::kDk) store_token<T, DP>((T *)z.dk.row(b, j, kh), z.D, key.dk, KS::k_factor(z, unit));
    if constexpr (KS::kDv) store_token<T, DP>((T *)z.dv.row(b, j, kh), z.D, key.dv, KS::v_factor());
  }
  bool bad[2] = {false, false};
  if constexpr (KS::kDv) bad[0] = any_not_finite(key.dv);
  if constexpr (KS::kDk) bad[1] = any_not_finite(key.dk);
  for (int of_k = 0; of_k < 2; ++of_k) {
    uint64_t rows = __ballot(either_half(of_k ? bad[1] : bad[0]) && key.seen.count > 0) & 0xffffffffu;
    if (rows) rows_written();
    while (rows) {
      const int r = __builtin_ctzll(rows);
      rows &= rows - 1;
      dkv_again<T>(z, s, b, kh, tile * kQueries + wave * 32 + r, of_k == 1);
    }
  }
}

// dk and dv of the sinks: 32 keys, which all wavefronts hold, against a share of all queries, of which each wavefront walks its own
// (a tile of 128 keys with a few sinks would have three of four wavefronts idle most of the way).  Reading q and do once more bounds
// it: 4 x 4112 tokens of 20 heads of 64 in bfloat16 21 us, 4 TB/s.
template <typename T, int DP, int PARTS> __global__ __launch_bounds__((64 * Few<T, DP>::kWaves), 1) void window_sink_kernel(const WindowArgs a) {
  using W = Few<T, DP>;
  using KS = KeySide<T, DP, PARTS>;
  constexpr int kWaves = W::kWaves;
  __shared__ __attribute__((aligned(16))) char tiles[kWaves * 2 * W::kStage];
  __shared__ __attribute__((aligned(16))) float lses[kWaves * 2 * 64], deltas[kWaves * 2 * 64];
  const int item = work_item(a);
  if (item >= a.items) return;
  const int rest = div_by(item, a.by_sink_parts), share = item - rest * a.sink_parts, bk = div_by(rest, a.by_sink_sets), set = rest - bk * a.sink_sets;
  const int b = div_by(bk, a.by_K), kh = bk - b * a.K;
  const Sample s = sample_of(a, b);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), j = set * 32 + (lane & 31);
  KS key;
  key.clear();
  key.seen = j < a.sinks ? seen_of(a, s, j) : Seen{0, 0};
  key.c = a.scale_log2;
  float unit = 1.0f;
  int top = (set + 1) * 32 < s.n ? (set + 1) * 32 : s.n;
  top = top < a.sinks ? top : a.sinks;
  const Queries range = queries_of(a, s, set * 32, top, true);
  if (range.from <= range.to) {
    const int first = range.from / 32, tiles_of = range.to / 32 - first + 1, steps = tiles_of * a.group, to = range.to;
    const int begin = share_begin(a.by_sink_parts, steps, share) + wave, end = share_begin(a.by_sink_parts, steps, share + 1);
    if constexpr (__is_same(T, f16_t)) {
      float most = 0.0f;
      for (int st = begin; st < end; st += kWaves) {
        const int64_t rows = ((int64_t)b * a.H + kh * a.group + st / tiles_of) * a.L;
        const int i = (first + st % tiles_of) * 32 + (lane & 31);
        if (i >= range.from && i <= to) most = fmaxf(most, load_global<float>(a.largest + rows + i));
      }
      unit = gradient_unit<T>(wave_max(most));
    }
    key.lowering = unit * (1.0f / 128.0f);
    key.load(a, b, j < s.n ? j : s.n - 1, kh);
    TilePair<T, DP, 32, 64> copy;
    copy.init(a.D, a.q.token_bytes, a.dout.token_bytes, to);
    LaneOffsets<T, DP> at;
    at.init(a.D);
    const unsigned lds = lds_address(tiles) + wave * 2 * W::kStage, lds_lse = lds_address(lses) + wave * 512, lds_delta = lds_address(deltas) + wave * 512;
    key.settle_operands();
    auto issue = [&](Step w, int buffer) {
      const int h = kh * a.group + w.g, i0 = (first + w.t) * 32;
      copy.go_to((const char *)a.q.row(b, 0, h), (const char *)a.dout.row(b, 0, h), i0);
      copy.issue(lds + buffer * W::kStage, W::kStage / 2);
      const unsigned r = (unsigned)(lane < to - i0 ? lane : to - i0) * 4;
      const int64_t row = ((int64_t)b * a.H + h) * a.L + i0;
      copy_to_lds<4>(uniform((const char *)(a.lse + row)), r, lds_lse + buffer * 256);
      copy_to_lds<4>(uniform((const char *)(a.delta + row)), r, lds_delta + buffer * 256);
    };
    Step step = {begin / tiles_of, begin % tiles_of}, next = step;
    int turn = 0;
    if (begin < end) issue(step, 0);
    for (int st = begin; st < end; st += kWaves) {
      const int now = turn;
      turn ^= 1;
      next.advance(kWaves, tiles_of);
      next_copies<2 * TileCopy<T, DP, 32, 64>::kCopies + 2>(st + kWaves < end, [&] { issue(next, turn); });
      char *qt = tiles + (wave * 2 + now) * W::kStage;
      key.template tile<32>(at, qt, qt + W::kStage / 2, lses + (wave * 2 + now) * 64, deltas + (wave * 2 + now) * 64, (first + step.t) * 32 + s.off);
      step = next;
    }
  }
  const WindowArgs &z = arguments_again();
  key.clear_unseen();
  // the wavefronts' sums, through the tiles' place
  float *mine = (float *)(tiles + wave * 2 * W::kStage);
  const int64_t slot = sink_slot(z, bk, set, share);
  auto add = [&](const auto &acc, float factor, float *to) {
    __syncthreads();  // (no copy is on its way: each wavefront has waited for its last one)
    #pragma unroll
    for (int x = 0; x < DP / 32; ++x)
#pragma unroll
      for (int r = 0; r < 16; r += 4)
        *(f32x4 *)(mine + (lane & 31) * W::kPitch + 32 * x + row_of(r, lane >> 5)) =
            f32x4{acc[x][r] * factor, acc[x][r + 1] * factor, acc[x][r + 2] * factor, acc[x][r + 3] * factor};
    __syncthreads();
    for (int e = threadIdx.x; e < 32 * DP / 4; e += 64 * kWaves) {
      const int r = e / (DP / 4), d = e % (DP / 4) * 4;
      if (d >= z.D) continue;
      f32x4 v = *(const f32x4 *)((const float *)tiles + r * W::kPitch + d);
#pragma unroll
      for (int n = 1; n < kWaves; ++n) v += *(const f32x4 *)((const float *)(tiles + n * 2 * W::kStage) + r * W::kPitch + d);
      store_global<f32x4>(to + (slot + r) * z.D + d, v);
    }
  };
  if constexpr (KS::kDk) add(key.dk, KS::k_factor(z, unit), z.part_k);
  if constexpr (KS::kDv) add(key.dv, KS::v_factor(), z.part_v);
}

// Sums of the keys that several workgroups shared, all keys or the sinks.
template <typename T> __global__ __launch_bounds__(kBlock) void window_sum_kernel(const WindowArgs a, const Joining of_sinks, const Joining of_others) {
  __shared__ int bad_k[kBlock], bad_v[kBlock], any_bad;
  __shared__ f32x4 place[kBlock];
  // (the first workgroups have the sinks, the others, if there are any, the other keys)
  const bool sink = (int)blockIdx.x < a.sink_blocks;
  const Joiner with(sink ? of_sinks : of_others);
  const int r = with.row, d = with.d, rows_here = with.rows_here;
  const int first = sink ? 0 : a.sinks, rows = sink ? a.sinks : a.S - a.sinks;
  bad_k[threadIdx.x] = bad_v[threadIdx.x] = 0;
  if (threadIdx.x == 0) any_bad = 0;
  const int block = (int)blockIdx.x - (sink ? 0 : a.sink_blocks), id = block * rows_here + r;
  const bool there = r < rows_here && id < (int64_t)a.B * a.K * rows;
  const int bk = (unsigned)id / (unsigned)rows, j = first + (id - bk * rows), b = div_by(bk, a.by_K), kh = bk - b * a.K;
  f32x4 k = {}, v = {};
  if (there) {
    const int64_t slot = sink ? sink_slot(a, bk, j / 32, 0) + j % 32 : tile_slot(a, bk, j / kQueries, 0) + j % kQueries;
    const int64_t at = slot * a.D + d, step = (int64_t)(sink ? 32 : kQueries) * a.D;
    const int parts = sink ? a.sink_parts : a.shares;
#pragma unroll 8
    for (int n = with.part; n < parts; n += with.joiners) {
      k += load_global<f32x4>(a.part_k + at + n * step);
      v += load_global<f32x4>(a.part_v + at + n * step);
    }
  }
  const auto add = [](f32x4 x, f32x4 y) { return x + y; };
  k = joined(with, k, place, add);
  v = joined(with, v, place, add);
  if (with.joiners == 1) __syncthreads();  // (bad is cleared)
  if (there && with.part == 0) {
    const float tk[4] = {k[0], k[1], k[2], k[3]}, tv[4] = {v[0], v[1], v[2], v[3]};
    using LV = LaneVec<T, 4>;
    LV::store((T *)a.dk.row(b, j, kh) + d, LV::pack(tk));
    LV::store((T *)a.dv.row(b, j, kh) + d, LV::pack(tv));
    if (!(k[0] * 0.0f + k[1] * 0.0f + k[2] * 0.0f + k[3] * 0.0f == 0.0f)) bad_k[r] = any_bad = 1;
    if (!(v[0] * 0.0f + v[1] * 0.0f + v[2] * 0.0f + v[3] * 0.0f == 0.0f)) bad_v[r] = any_bad = 1;
  }
  __syncthreads();
  if (!any_bad) return;
  rows_of_all_written();
  for (int n = threadIdx.x >> 6; n < rows_here; n += 4) {
    if (!(bad_k[n] | bad_v[n])) continue;
    const WindowArgs &z = arguments_again();
    const int row = block * rows_here + n;
    const int bk = (unsigned)row / (unsigned)rows, key = first + (row - bk * rows), b = div_by(bk, z.by_K), kh = bk - b * z.K;
    const Sample s = sample_of(z, b);
    if (seen_of(z, s, key).count == 0) continue;
    if (bad_v[n]) dkv_again<T>(z, s, b, kh, key, false);
    if (bad_k[n]) dkv_again<T>(z, s, b, kh, key, true);
  }
}

}  // namespace gn
