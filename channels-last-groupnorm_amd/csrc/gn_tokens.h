// Host-side interface of the operators for token streams: argument blocks shared by the C ABI (gn_tokens.hip) and the
// kernels' launchers (gn_rms.hip, gn_rotary.hip: compiled once per element type; gn_clip.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>
#include "../../include/gnnhwc_tokens.h"
#include "gn_plan.h"

namespace gn {

enum { GN_F8 = GNNHWC_F8E4M3, GN_I8 = GNNHWC_I8 };

// Rows of the norms: C channels as nvec lane vectors, dealt to lpr = 2^lpr_log2 lanes.
struct RowCut {
  int vec, nvec, lpr, lpr_log2, nv, threads;
  bool ragged;
};

struct RmsFwd {  // (see gn_rms.h)
  const void *x, *res, *w;
  void *sum, *y;
  float *scales;
  int64_t rows, x_stride, res_stride;
  double eps, inv_c;
  int C, nvec, lpr, lpr_log2;
  int block_lanes, nblocks, qtype;  // quantised: lanes per scale (0: one scale per row), scales per row, type
  float q_most;
};
struct RmsBwd {
  const void *dy, *ds, *s, *w;
  void *dx, *part;
  int64_t rows, dy_stride, ds_stride, s_stride;
  double eps, inv_c;
  int C, nvec, lpr, lpr_log2;
};

// How lanes share a head: channels of a lane vector; pairs near each other or far; one vector of a lane (a head's access is
// whole) or two.
struct RotaryCut {
  int vec;
  bool near, whole;
};
// Most heads of a token that a group of lanes turns; backward, most lane vectors of x (and as many of its gradient) that a lane holds.
constexpr int kRotaryHeads = 4, kRotaryBwdVecs = 4;
struct RotarySide {  // q or k
  const void *in, *grad, *weight;
  void *out;
  int64_t in_stride[3], grad_stride[3], out_stride[3];  // batch, token, head
  int heads, groups;  // groups of lanes that share a token's heads
};
struct RotaryArgs {
  RotarySide side[2];
  const void *pos;
  int64_t pos_stride[2];
  const float *freq;
  int pos_type, axes, ends[4], P, D;
  int nvec, lanes, lanes_log2;  // lanes that a head takes, lanes of a group
  int tokens, L, groups;        // batch * tokens, tokens of a sample, groups of a token (q's, then k's)
  int span;                     // most tokens that a workgroup's groups belong to
  Divisor by_groups, by_L, by_half;
  int walkers, token_step;      // backward behind a norm: groups that work, tokens between two of a group
  double eps, inv_d;
  float sign;                   // -1: turn back
  void *part;
};

// Sums of `count` rows of partial results, C values each, in a fixed order (gn_rms.h).
struct PartialSum {
  const void *part;
  void *out[2];  // columns below and from `split` on; null: not wanted
  int count, C, split, out_dtype;
};

constexpr int kMostChannels = 16384;
constexpr int kRowVectors = 3;  // most lane vectors of a row per lane, but for the longest rows
// What the memory-side cache is counted on to hold until the next kernel.  Inputs beyond it are read past the caches: backward of
// float16 (65536, 2560) 239 -> 233 us, its forward 220 -> 219; but forward of bf16 (90000, 320), which the cache can hold, 17.7 -> 20.1.
constexpr int64_t kCachedBytes = (int64_t)224 << 20;

#define GN_DECLARE_TOKENS(S)                                                                            \
  hipError_t launch_rms_fwd_##S(const RmsFwd &a, const RowCut &cut, int pdtype, bool quant, hipStream_t stream);   \
  hipError_t launch_rms_bwd_##S(const RmsBwd &a, const RowCut &cut, int pdtype, int blocks, void *dw, hipStream_t stream); \
  hipError_t launch_rotary_##S(const RotaryArgs &a, const RotaryCut &cut, bool norm, int pdtype, hipStream_t stream);         \
  hipError_t launch_rotary_norm_bwd_##S(const RotaryArgs &a, const RotaryCut &cut, int pdtype, int blocks, void *const (&dw)[2], hipStream_t stream);
// Gradients of one launch; the whole table travels as a kernel argument.
struct ClipEntry {
  const void *in;
  void *out;
  int64_t n;
  unsigned first_chunk;
  int types;  // dtype | out dtype << 8
};
constexpr int kClipEntries = 112;
struct ClipTable {
  ClipEntry e[kClipEntries];
  int count;
  unsigned chunks;
};
constexpr int kClipChunk = 16384;   // elements
constexpr int kClipBlocks = 1024;   // workgroups of a norm's launch, each with a partial sum
constexpr int kClipTables = 4;       // tables whose partial sums every workgroup of the second pass adds itself
struct ClipFinish {
  const double *part;
  int parts;
  double max_norm, eps, grad_scale;
  void *total;
  int total_dtype;
  bool in_place;
};
hipError_t launch_clip_norm(const ClipTable &t, double *part, int blocks, hipStream_t stream);
hipError_t launch_clip_sum(double *part, int parts, hipStream_t stream);
hipError_t launch_clip_apply(const ClipTable &t, const ClipFinish &f, bool streams, int blocks, hipStream_t stream);

GN_DECLARE_TOKENS(f32)
GN_DECLARE_TOKENS(f64)
GN_DECLARE_TOKENS(f16)
GN_DECLARE_TOKENS(bf16)
#undef GN_DECLARE_TOKENS

}  // namespace gn
