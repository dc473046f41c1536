/*
 * gnnhwc_tokens.h -- the second part of the C ABI of libgnnhwc_hip.so (see gnnhwc.h): operators for token streams, i.e. for
 * the transformer blocks that stand between channels-last features in image and video models, in training and in serving.
 * The reference has no counterpart to any of them.
 *
 *   gnnhwc_rms_*       root-mean-square norm of rows, with the residual's addition in front, forward and backward, and with
 *                      results in 8 bits with scales
 *   gnnhwc_rotary*     rotary positions with several axes on q and k, optionally behind a norm of each head
 *   gnnhwc_clip        the norm over many gradients and their clipping
 *   gnnhwc_window_*    softmax attention in which a token sees a window around it and a few first tokens, forward, backward, and
 *                      of the newest tokens against what a cache holds
 *   gnnhwc_dropout     dropout from a counter-based generator, with the residual's addition
 *
 * Conventions are those of gnnhwc.h: device pointers on the current device, asynchronous on `stream`, no synchronisation, no
 * allocation, a caller-provided workspace whose contents on entry are ignored (8-byte aligned is enough here, but for the attention's:
 * GNNHWC_WINDOW_WORKSPACE_ALIGNMENT), GNNHWC_OK or a negative code with the message in gnnhwc_last_error(), and nothing launched when
 * an error is returned.  All of them may be captured into a HIP graph; all results are reproducible bit for bit.  These operators
 * keep no state between calls.  Tensors need the alignment of their element only (the attention's: see there).  Outputs must not
 * overlap inputs unless stated.
 */
#ifndef GNNHWC_TOKENS_H
#define GNNHWC_TOKENS_H

#include "gnnhwc.h"

#ifdef __cplusplus
extern "C" {
#endif

/* 8-bit result types, besides the dtype codes of gnnhwc.h */
enum {
  GNNHWC_F8E4M3 = 4, /* OCP e4m3 (finite values to 448, no infinities) */
  GNNHWC_I8 = 5      /* -127 .. 127 */
};

/*
 * Root-mean-square norm.  Rows of C channels (1 <= C <= 16384; 8192 for GNNHWC_F64), row i of x at x + i * x_stride elements:
 *   s = x + residual, rounded to dtype once;  y = s / sqrt(mean(s^2) + eps) * weight
 * with the mean, the root and the products in float32 (float64 for F64 data) and one rounding at the end.
 *   residual : rows like x's, residual_stride apart, or NULL.
 *   weight   : C values in param_dtype (dtype, or GNNHWC_F32 for F16 / BF16 data), or NULL (1).
 *   sum_out  : receives s, rows of C contiguous; NULL where nobody needs it.  Only with a residual.
 *   y        : rows of C contiguous.
 */
int gnnhwc_rms_fwd(const void *x, const void *residual, const void *weight, void *sum_out, void *y,
                   int64_t rows, int64_t C, int64_t x_stride, int64_t residual_stride,
                   double eps, int dtype, int param_dtype, void *stream);

/*
 * The same with y in 8 bits, rounded from the float32 result:  per block of `block` consecutive channels of a row
 *   scale = max(max |y| / most, 2^-126),  q = round to nearest even(y / scale)       most = 448 (F8E4M3), 127 (I8)
 *   block  : a power of two from 16 to 256, the last block of a row may be shorter; 0 or any value >= C: one scale per row.
 *   q      : (rows, C);  scales : float (rows, ceil(C / block)).
 * A row with a NaN or an infinity in it gets NaN scales (in the blocks that they reach) and, as F8E4M3, NaN values.
 * dtype: F32, F16 or BF16.
 */
int gnnhwc_rms_fwd_quant(const void *x, const void *residual, const void *weight, void *sum_out, void *q, float *scales,
                         int64_t rows, int64_t C, int64_t x_stride, int64_t residual_stride, int64_t block,
                         double eps, int dtype, int param_dtype, int q_dtype, void *stream);

/*
 * Backward of gnnhwc_rms_fwd.  s: its input (its sum_out where it had a residual).  With r = 1 / sqrt(mean(s^2) + eps), which is
 * computed again, g = dy * weight and h = s * r:
 *   dx = r * (g - h * mean(g * h)) + ds        the gradient of x and of residual alike
 *   dweight = sum over rows of dy * h          in param_dtype, summed in float32 (float64 for F64) in a fixed order
 *   ds      : gradient of sum_out, or NULL.
 *   dweight : NULL to skip it.     dx : rows of C contiguous; NULL to skip it.
 */
size_t gnnhwc_rms_bwd_workspace_bytes(int64_t rows, int64_t C, int dtype);
int gnnhwc_rms_bwd(const void *dy, const void *ds, const void *s, const void *weight, void *dx, void *dweight,
                   int64_t rows, int64_t C, int64_t dy_stride, int64_t ds_stride, int64_t s_stride,
                   double eps, int dtype, int param_dtype, void *workspace, size_t workspace_bytes, void *stream);

/*
 * Rotary positions.  A head's first 2 P channels are P pairs, pair j being channels (2j, 2j + 1) if `interleaved`, else
 * (j, j + P); the channels behind them stay as they are.  Pair j belongs to axis a = the first with j < section_end[a],
 * P = section_end[axes - 1], and is turned by the angle position[a] * frequencies[j]:
 *   (u, v) -> (u cos - v sin, u sin + v cos)
 * The angle is formed and reduced with more than 32 bits, so that long positions lose nothing.  With q_weight / k_weight a
 * head is first normalised over all its channels, t / sqrt(mean(t^2) + eps) * weight; one rounding at the end.
 * Strides are in elements; channels of a head are contiguous.
 *
 * Forward: reads q and k, writes q_out and k_out.
 * Backward (gnnhwc_rotary_bwd): q_grad and k_grad are the gradients of the forward's outputs, q_out and k_out receive those of
 * q and k; q and k are read only where there is a weight, whose gradient goes to q_dweight / k_dweight (NULL to skip).
 * k (with kv_heads = 0) may be absent.  An output may be the buffer of the input it replaces, with the same strides (q_out
 * that of q, or of q_grad in the backward).
 */
typedef struct gnnhwc_rotary_call {
  const void *q, *k, *q_grad, *k_grad;
  void *q_out, *k_out;
  int64_t q_stride[3], k_stride[3];             /* batch, token, head */
  int64_t q_grad_stride[3], k_grad_stride[3];
  int64_t q_out_stride[3], k_out_stride[3];
  int64_t batch, tokens, heads, kv_heads;
  int64_t head_dim;                             /* even, 2 .. 256; above 128 a multiple of 8, as is 2 P then */
  int64_t axes, section_end[4];                 /* 1 .. 4 axes, their ends ascending */
  int64_t interleaved;
  const void *positions;                        /* (batch, tokens, axes), axes contiguous */
  int64_t position_stride[2];                   /* batch (0: the same for all), token */
  int64_t position_type;                        /* 0 int32, 1 int64 (within 32 bits), 2 float; exact up to 2^24 */
  const float *frequencies;                     /* P */
  const void *q_weight, *k_weight;              /* both or none (k_weight only with k) */
  void *q_dweight, *k_dweight;
  double eps;
  int64_t dtype, param_dtype;
} gnnhwc_rotary_call;

int gnnhwc_rotary(const gnnhwc_rotary_call *call, void *stream);
size_t gnnhwc_rotary_bwd_workspace_bytes(const gnnhwc_rotary_call *call);
int gnnhwc_rotary_bwd(const gnnhwc_rotary_call *call, void *workspace, size_t workspace_bytes, void *stream);

/*
 * The Euclidean norm over `count` tensors (any dtype codes of gnnhwc.h, mixed, each n[i] contiguous elements) and their clipping:
 *   total = |grad_scale| * sqrt(sum of squares)                     written to `total` (float; double if total_dtype is F64)
 *   out[i] = in[i] * (grad_scale * min(1, max_norm / (total + eps)))
 * Squares are summed in float64.  grad_scale: 1, or the reciprocal of a loss scale.  A total that is NaN gives NaN.
 *   out : NULL: in place (nothing is written where the factor is 1); else per tensor where it goes, in out_dtype[i].
 *         out[i] may be in[i] where the types are the same; no other two tensors of which one is written may overlap.
 *   max_norm : infinity for no bound;  out NULL, grad_scale 1 and an infinite max_norm compute the norm only.
 * The arrays are host memory and are not read after the call returns.
 */
size_t gnnhwc_clip_workspace_bytes(int64_t count);
int gnnhwc_clip(const void *const *in, void *const *out, const int64_t *n, const int *dtype, const int *out_dtype,
                int64_t count, double max_norm, double eps, double grad_scale, void *total, int total_dtype,
                void *workspace, size_t workspace_bytes, void *stream);

/*
 * Softmax attention of `heads` query heads over `kv_heads` key heads (a divisor; head h goes with key head h / (heads / kv_heads)):
 *   s_ij = scale q_i . k_j,   out_i = sum_j softmax_j(s_ij) v_j   over the keys j that query i sees.
 * A sample has n keys: `keys`, or its entry of `lengths` (clamped to 0 .. keys).  Query i stands at place p = i + keys - tokens,
 * or with `at_end` at i + n - tokens: the queries are the newest of the sample's own tokens.  It sees key j < n if
 * |p - j| <= window or j < sinks, and, if `causal`, j <= p.  A query whose p is not among 0 .. n - 1, or that sees nothing, gets
 * zeros; what lies behind n in k and v is not read, in q and out_grad has no effect, and gets zeros for gradients.  An infinity or a NaN reaches
 * only the tokens that see it.
 * Scores, softmax and sums are in float32; softmax weights (and in the backward their derivatives) are rounded to dtype
 * once, as operands of the second product.  dtype: F32, F16 or BF16.  F16 has small ones in fixed steps: weights are off by up to
 * 2^-25 of their query's largest (in v_grad 2^-37 of one), the derivatives by up to 2^-29 of the largest |out_grad| of the query or,
 * in k_grad, of the queries that a workgroup visits.
 *   lse      : float (batch, heads, tokens): log2 of the softmax's sum, infinite for a query that sees nothing.  Written by the
 *              forward unless NULL, read by the backward.
 *   out_rest : (batch, tokens, heads, head_dim) of dtype, no gaps, 16-byte aligned: what rounding left of out.  Written by the forward
 *              and read by the backward unless NULL; F32 has none.  Without it gradients of queries that see a few tokens are less
 *              exact (they are differences that the rounding of out is large against).
 *   strides  : of batch, token and head in elements, each a whole multiple of 16 bytes (but for dimensions of size 1), as are the
 *              addresses; a token's below 2^25 bytes.  Channels of a head are contiguous.
 * Backward (not with at_end): reads q, k, v, out, out_grad, lse and out_rest, writes q_grad, k_grad and v_grad.
 * Outputs must not overlap inputs or each other.
 */
typedef struct gnnhwc_window_call {
  const void *q, *k, *v;        /* (batch, tokens, heads, head_dim), (batch, keys, kv_heads, head_dim) twice */
  void *out;                    /* like q; read by the backward */
  float *lse;
  void *out_rest;               /* or NULL */
  const void *out_grad;
  void *q_grad, *k_grad, *v_grad;
  int64_t q_stride[3], k_stride[3], v_stride[3], out_stride[3];
  int64_t out_grad_stride[3], q_grad_stride[3], k_grad_stride[3], v_grad_stride[3];
  int64_t batch, tokens, keys, heads, kv_heads;
  int64_t head_dim;             /* a multiple of 8, to 256 (F32: 128) */
  int64_t window;               /* -1: no bound */
  int64_t sinks, causal;
  const void *lengths;          /* batch values, or NULL */
  int64_t length_type;          /* 0 int32, 1 int64 */
  int64_t at_end;
  double scale;                 /* positive */
  int64_t dtype;
} gnnhwc_window_call;

/* What gnnhwc_window_workspace_bytes returns for a call that needs none: its workspace may be NULL.  (The backward's may not.) */
#define GNNHWC_WINDOW_NO_WORKSPACE ((size_t)256)
/* What the address of these functions' workspace is a whole multiple of (it holds rows that are read 16 bytes at a time). */
#define GNNHWC_WINDOW_WORKSPACE_ALIGNMENT ((size_t)16)
size_t gnnhwc_window_workspace_bytes(const gnnhwc_window_call *call);
int gnnhwc_window(const gnnhwc_window_call *call, void *workspace, size_t workspace_bytes, void *stream);
size_t gnnhwc_window_bwd_workspace_bytes(const gnnhwc_window_call *call);
int gnnhwc_window_bwd(const gnnhwc_window_call *call, void *workspace, size_t workspace_bytes, void *stream);

/*
 * Dropout:  y[e] = (kept ? x[e] f : 0) + residual[e],  f = 1 / (1 - p'),  for e in 0 .. n - 1, in float32 (float64 for F64) and rounded to
 * dtype once.  f is rounded to float32 (float64) itself, so that of F32 and F64 the product is off by a unit in the last place or less.
 * p' is p in whole multiples of 2^-16, rounded to nearest.  Element e is kept if its 16 random bits are at least 65536 p': they are
 * half e % 2 (the lower first) of word (e / 2) % 4 of Philox 4x32 with 7 rounds, whose counter is (e / 8, offset), both 64 bits, the
 * lower word first, and whose key is the seed.  The same seed and offset give the same bits: the backward is this call on the gradient, without a
 * residual.  What is dropped has no effect, an infinity or a NaN neither.
 *   residual : NULL for none.    y : may be x, or residual.
 *   seed_at  : device memory that holds the seed when the kernel runs (so that a captured graph's replays differ), or NULL.
 */
int gnnhwc_dropout(const void *x, const void *residual, void *y, int64_t n, double p, uint64_t seed, const int64_t *seed_at,
                   uint64_t offset, int dtype, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* GNNHWC_TOKENS_H */
