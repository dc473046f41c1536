// C ABI of the operators for token streams (declared in include/gnnhwc_tokens.h): argument checks, launch planning,
// element-type dispatch.
#include <hip/hip_runtime.h>
#include <math.h>

#include <algorithm>
#include <vector>

#include "gn_error.h"
#include "gn_tokens.h"

namespace gn {
namespace {

int elem_size(int64_t dtype) {
  switch (dtype) {
    case GN_F32: return 4;
    case GN_F64: return 8;
    case GN_F16: return 2;
    case GN_BF16: return 2;
    default: return 0;
  }
}
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int log2_of(int v) {
  int l = 0;
  while ((1 << l) < v) ++l;
  return l;
}
int invalid(const char *what) { return fail(GNNHWC_ERR_INVALID_ARGUMENT, "%s", what); }
int launched(hipError_t e, const char *what) {
  return e == hipSuccess ? GNNHWC_OK : fail(GNNHWC_ERR_LAUNCH, "%s: %s", what, hipGetErrorString(e));
}

int check_types(int64_t dtype, int64_t param_dtype) {
  if (!elem_size(dtype)) return fail(GNNHWC_ERR_INVALID_ARGUMENT, "unknown dtype code %lld", (long long)dtype);
  const bool half = dtype == GN_F16 || dtype == GN_BF16;
  if (param_dtype != dtype && !(half && param_dtype == GN_F32))
    return fail(GNNHWC_ERR_INVALID_ARGUMENT, "weight dtype %lld does not go with dtype %lld (the same, or f32 for 16-bit data)",
                (long long)param_dtype, (long long)dtype);
  return GNNHWC_OK;
}
int check_rows(int64_t rows, int64_t C, int dtype, int param_dtype) {
  if (const int rc = check_types(dtype, param_dtype)) return rc;
  const int64_t most = dtype == GN_F64 ? kMostChannels / 2 : kMostChannels;
  if (C < 1 || C > most)
    return fail(GNNHWC_ERR_INVALID_ARGUMENT, "rows of %lld channels: 1 to %lld are supported", (long long)C, (long long)most);
  if (rows < 0 || rows > 0x7fffffff)
    return fail(GNNHWC_ERR_INVALID_ARGUMENT, "%lld rows: 0 to 2^31 - 1 are supported", (long long)rows);
  return GNNHWC_OK;
}
// (eps may be zero: a row of zeros then gives NaN, as the formula does)
int check_eps(double eps) { return eps >= 0 && eps < INFINITY ? GNNHWC_OK : invalid("eps must be finite and not negative"); }

// A launch has fewer than 2^32 threads: calls with more rows than that go out in pieces.
int64_t rows_per_launch(const RowCut &cut) { return ((int64_t)1 << 31) / cut.lpr; }

#define GN_BY_TYPE(dtype, call)                 \
  ((dtype) == GN_F32   ? call(f32)              \
   : (dtype) == GN_F64 ? call(f64)              \
   : (dtype) == GN_F16 ? call(f16)              \
                       : call(bf16))

RmsFwd fwd_args(const void *x, const void *residual, const void *weight, void *sum_out, void *y, int64_t rows, int64_t C,
                int64_t x_stride, int64_t residual_stride, double eps, const RowCut &cut) {
  RmsFwd a = {};
  a.x = x; a.res = residual; a.w = weight;
  a.sum = sum_out; a.y = y;
  a.rows = rows; a.x_stride = x_stride; a.res_stride = residual_stride;
  a.eps = eps; a.inv_c = 1.0 / (double)C;
  a.C = (int)C; a.nvec = cut.nvec; a.lpr = cut.lpr; a.lpr_log2 = cut.lpr_log2;
  return a;
}
int launch_fwd(RmsFwd a, const RowCut &cut, int dtype, int param_dtype, bool quant, hipStream_t stream, const char *what) {
  const int64_t rows = a.rows, most = rows_per_launch(cut), es = elem_size(dtype);
  for (int64_t at = 0; at < rows; at += most) {
    a.rows = std::min(most, rows - at);
#define GN_CALL(S) launch_rms_fwd_##S(a, cut, param_dtype, quant, stream)
    if (const hipError_t e = GN_BY_TYPE(dtype, GN_CALL)) return launched(e, what);
#undef GN_CALL
    a.x = (const char *)a.x + most * a.x_stride * es;
    if (a.res) a.res = (const char *)a.res + most * a.res_stride * es;
    if (a.sum) a.sum = (char *)a.sum + most * a.C * es;
    a.y = (char *)a.y + most * a.C * (quant ? 1 : es);
    if (a.scales) a.scales += most * a.nblocks;
  }
  return GNNHWC_OK;
}
int check_fwd(const void *x, const void *residual, void *sum_out, const void *y, int64_t rows) {
  if (rows > 0 && (!x || !y)) return invalid("null tensor");
  if (sum_out && !residual) return invalid("sum_out without a residual");
  return GNNHWC_OK;
}

// How a row's lane vectors are dealt to lanes: the fewest lanes (a power of two) that leave none more than three (against five:
// bf16 in 8 bits (280000, 200) 36 and 50 us, (16384, 2560) with 128 channels a block 53 and 55; backward of bf16 (140000, 200) 34
// and 38; of float16 (65536, 2560) 233 and 229, its forward 219 either way).
// `whole`: rows that are not whole lines of memory in one access each, up to a wavefront, where several would write parts of
// lines (forward, bf16 (140000, 200) with a residual 57 -> 39 us, (966103, 80) 102 -> 61; rows of whole lines lose by it,
// (90000, 320) 17.7 -> 19.9, as do the backward, (140000, 200) 34 -> 46, whose few workgroups want more of each row on its way,
// and 8 bits, (280000, 200) 36 -> 47).
RowCut rms_cut(int64_t C, int esize, int least_lanes, bool whole) {
  const int vec = 16 / esize;
  RowCut c;
  c.vec = C < vec ? 1 : vec;
  c.nvec = (int)ceil_div(C, c.vec);
  c.ragged = C % c.vec != 0;
  c.lpr = std::max(8, least_lanes);
  if (whole && C * esize % 128 != 0)
    while (c.lpr < 64 && c.nvec > c.lpr) c.lpr <<= 1;
  // (two where a workgroup is wider than 256: a third does not fit the registers of 1024 threads in the backward)
  while (c.lpr < 1024 && c.nvec > (c.lpr > 256 ? 2 : kRowVectors) * c.lpr) c.lpr <<= 1;
  c.nv = (int)ceil_div(c.nvec, c.lpr);
  c.lpr_log2 = log2_of(c.lpr);
  c.threads = c.lpr > 256 ? c.lpr : 256;
  return c;
}
// Workgroups of the backward's walk: as many as walk equally far, up to two per CU (with three or four, float16 (65536, 2560)
// takes 240 and 262 us instead of 233; bf16 (16384, 1280) 33.5 and 37.7 instead of 34.9, (140000, 200) 31 and 32 instead of 34,
// but each leaves a partial row to write and to add).
int rms_bwd_blocks(int64_t rows, const RowCut &cut) {
  const int64_t steps = ceil_div(rows, cut.threads / cut.lpr);
  return steps == 0 ? 0 : (int)ceil_div(steps, ceil_div(steps, 2 * kNumCU));
}

// ---- rotary ----
struct RotaryPlan {
  RotaryArgs a;
  RotaryCut cut;
  int blocks;  // of the backward behind a norm
  bool empty;
};
int64_t partial_bytes(const RotaryPlan &p, int64_t dtype) {
  return (int64_t)p.blocks * 2 * p.a.D * (dtype == GN_F64 ? 8 : 4);
}

int plan_rotary(const gnnhwc_rotary_call *c, bool backward, RotaryPlan &p) {
  if (!c) return invalid("null call");
  if (const int rc = check_types(c->dtype, c->q_weight ? c->param_dtype : c->dtype)) return rc;
  if (c->batch < 0 || c->tokens < 0 || c->heads < 1 || c->kv_heads < 0) return invalid("batch, tokens or heads out of range");
  if (c->heads > 65535 || c->kv_heads > 65535) return invalid("heads out of range: at most 65535");
  if (c->head_dim < 2 || c->head_dim > 256 || c->head_dim % 2) return invalid("head_dim must be even and 2 to 256");
  if (c->axes < 1 || c->axes > 4) return invalid("1 to 4 axes are supported");
  int64_t last = 0;
  for (int i = 0; i < c->axes; ++i) {
    if (c->section_end[i] < last) return invalid("section_end must not descend");
    last = c->section_end[i];
  }
  if (last < 1 || 2 * last > c->head_dim) return invalid("sections must hold 1 to head_dim / 2 pairs");
  if (c->position_type < 0 || c->position_type > 2) return invalid("position_type must be 0 (int32), 1 (int64) or 2 (float)");
  if (c->tokens > 0 && c->batch > 0x40000000 / c->tokens) return invalid("too many tokens: at most 2^30");
  if ((c->kv_heads > 0) != (c->k_out != nullptr) && c->batch * c->tokens > 0) return invalid("kv_heads without k_out, or the reverse");
  if (c->kv_heads > 0 && (c->q_weight != nullptr) != (c->k_weight != nullptr)) return invalid("q_weight and k_weight go together");
  const bool norm = c->q_weight != nullptr;
  if (const int rc = check_eps(norm ? c->eps : 0)) return rc;
  p = {};
  RotaryArgs &a = p.a;
  p.empty = c->batch == 0 || c->tokens == 0;
  a.D = (int)c->head_dim;
  a.P = (int)last;
  const int half = a.D / 2, most = c->dtype == GN_F64 ? 2 : c->dtype == GN_F32 ? 4 : 8;
  // The widest lane vector that divides what it has to; half of 16 bytes for half-precision heads such as 40 with far pairs.
  // Whole heads (PairLane, gn_rotary.h) for 16 bits:
  // - near pairs, always: (16384, 20 + 20, 64) 31 us, in halves 36; (65536, 8 + 8, 80) 59 and 72; (74800, 24 + 24, 64) 153 and
  //   178; behind a norm backward 47 and 65, 121 and 116.  Of 32 bits halves are longer and a workgroup of half as many heads costs
  //   more: (308142, 2 + 1, 96) whole 140, in halves 127; (770, 24 + 12, 40) 5.0 and 4.3.
  // - far pairs, forward, where they fill three quarters of the lanes: (16384, 20 + 20, 64) 32 us, in halves 36.5; (46800,
  //   24 + 24, 96) 149 and 183; of 160 channels, 20 of 32 lanes, (13000, 5 + 1) 15.3 and 12.5.  Behind a norm backward: 50 and 50,
  //   (13770, 12 + 2, 80) 30 and 24.7.
  const bool bits16 = c->dtype == GN_F16 || c->dtype == GN_BF16, near = c->interleaved != 0;
  const int vecs16 = a.D / 8;
  const bool far_whole = bits16 && !near && !(backward && norm) && a.D % 8 == 0 && a.P % 8 == 0 && 4 * vecs16 >= 3 << log2_of(vecs16);
  const bool wide = far_whole || (bits16 && near);
  int vec = 1;
  for (int s = most; s > 1; s >>= 1)
    if (!(s == 2 && most != 2) && (wide ? a.D : half) % s == 0 && (near || a.P % s == 0)) {
      vec = s;
      break;
    }
  p.cut = {vec, near, wide && vec > 1};
  const int vecs = p.cut.whole ? 1 : 2;
  a.nvec = a.D / (vecs * vec);
  if (a.nvec > 64) return invalid("heads of more than 128 channels must have a multiple of 8 channels, and so must their pairs");
  a.lanes_log2 = log2_of(a.nvec);
  a.lanes = 1 << a.lanes_log2;
  if (p.empty) return GNNHWC_OK;

  const int64_t tokens = c->batch * c->tokens;
  if (!c->positions || !c->frequencies) return invalid("null positions or frequencies");
  if (!c->q_out || (c->kv_heads && !c->k_out)) return invalid("null output");
  const bool reads = !backward || norm;
  if (reads && (!c->q || (c->kv_heads && !c->k))) return invalid("null tensor");
  if (backward && (!c->q_grad || (c->kv_heads && !c->k_grad))) return invalid("null gradient");
  const int64_t heads[2] = {c->heads, c->kv_heads};
  // Heads that a group turns: as many as it has registers for, each of them on its way at once, as long as the groups fill the
  // device four times.
  int take = backward && norm ? kRotaryBwdVecs / vecs : kRotaryHeads;
  while (take > 1 && tokens * (ceil_div(heads[0], take) + ceil_div(heads[1], take)) * a.lanes < (int64_t)4 * kNumCU * kBlock) take >>= 1;
  const void *in[2] = {c->q, c->k}, *grad[2] = {c->q_grad, c->k_grad}, *weight[2] = {c->q_weight, c->k_weight};
  void *out[2] = {c->q_out, c->k_out};
  const int64_t *is[2] = {c->q_stride, c->k_stride}, *gs[2] = {c->q_grad_stride, c->k_grad_stride}, *os[2] = {c->q_out_stride, c->k_out_stride};
  for (int i = 0; i < 2; ++i) {
    RotarySide &s = a.side[i];
    const bool turns_grad = backward && !norm;  // the gradient is what is turned
    s.in = turns_grad ? grad[i] : in[i];
    s.grad = grad[i];
    s.weight = weight[i];
    s.out = out[i];
    for (int d = 0; d < 3; ++d) {
      s.in_stride[d] = turns_grad ? gs[i][d] : is[i][d];
      s.grad_stride[d] = gs[i][d];
      s.out_stride[d] = os[i][d];
    }
    s.heads = (int)heads[i];
    s.groups = (int)ceil_div(heads[i], take);
  }
  a.groups = a.side[0].groups + a.side[1].groups;
  if (tokens * a.groups > 0x7fff0000 || tokens * a.groups * a.lanes > 0xffff0000) return invalid("too many tokens and heads for one call");
  a.pos = c->positions;
  a.pos_stride[0] = c->position_stride[0];
  a.pos_stride[1] = c->position_stride[1];
  a.freq = c->frequencies;
  a.pos_type = (int)c->position_type;
  a.axes = (int)c->axes;
  for (int i = 0; i < 4; ++i) a.ends[i] = (int)(i < c->axes ? c->section_end[i] : last);
  a.tokens = (int)tokens;
  a.L = (int)c->tokens;
  a.by_groups = make_divisor(a.groups, 0);
  a.by_L = make_divisor(a.L, 0);
  a.by_half = make_divisor(half, 0);
  const int subs = kBlock / a.lanes;
  a.span = (int)std::min<int64_t>(tokens, (subs - 1 + a.groups - 1) / a.groups + 1);
  a.eps = c->eps;
  a.inv_d = 1.0 / a.D;
  a.sign = backward ? -1.0f : 1.0f;
  if (backward && norm) {
    // A walk of whole sets of groups, alike in length: at most three workgroups per CU (with four bf16 (16384, 20 + 20, 64) takes
    // 59 us instead of 47, float16 (65536, 8 + 8, 80) 132 instead of 121), or four where that spares the second turn.
    const int64_t steps = std::max<int64_t>(1, 3 * kNumCU * subs / a.groups);
    const int64_t turns = tokens <= steps + steps / 3 ? 1 : ceil_div(tokens, steps);
    a.token_step = (int)ceil_div(tokens, turns);
    a.walkers = a.token_step * a.groups;
    p.blocks = (int)ceil_div(a.walkers, subs);
  }
  return GNNHWC_OK;
}

}  // namespace
}  // namespace gn

using namespace gn;

extern "C" {

int gnnhwc_rms_fwd(const void *x, const void *residual, const void *weight, void *sum_out, void *y, int64_t rows, int64_t C,
                   int64_t x_stride, int64_t residual_stride, double eps, int dtype, int param_dtype, void *stream) {
  if (const int rc = check_rows(rows, C, dtype, weight ? param_dtype : dtype)) return rc;
  if (const int rc = check_eps(eps)) return rc;
  if (const int rc = check_fwd(x, residual, sum_out, y, rows)) return rc;
  if (rows == 0) return GNNHWC_OK;
  const RowCut cut = rms_cut(C, elem_size(dtype), 8, true);
  RmsFwd a = fwd_args(x, residual, weight, sum_out, y, rows, C, x_stride, residual_stride, eps, cut);
  return launch_fwd(a, cut, dtype, weight ? param_dtype : dtype, false, (hipStream_t)stream, "gnnhwc_rms_fwd");
}

int gnnhwc_rms_fwd_quant(const void *x, const void *residual, const void *weight, void *sum_out, void *q, float *scales,
                         int64_t rows, int64_t C, int64_t x_stride, int64_t residual_stride, int64_t block, double eps, int dtype,
                         int param_dtype, int q_dtype, void *stream) {
  if (const int rc = check_rows(rows, C, dtype, weight ? param_dtype : dtype)) return rc;
  if (dtype == GN_F64) return invalid("8-bit results take f32, f16 or bf16 data");
  if (q_dtype != GNNHWC_F8E4M3 && q_dtype != GNNHWC_I8) return fail(GNNHWC_ERR_INVALID_ARGUMENT, "unknown 8-bit type %d", q_dtype);
  if (const int rc = check_eps(eps)) return rc;
  if (const int rc = check_fwd(x, residual, sum_out, q, rows)) return rc;
  if (rows > 0 && !scales) return invalid("null scales");
  const bool by_row = block == 0 || block >= C;
  if (!by_row && (block < 16 || block > 256 || (block & (block - 1))))
    return fail(GNNHWC_ERR_INVALID_ARGUMENT, "a block of %lld channels: a power of two from 16 to 256, or 0 for whole rows", (long long)block);
  if (rows == 0) return GNNHWC_OK;
  const int lanes = by_row ? 0 : (int)block / (16 / elem_size(dtype));
  const RowCut cut = rms_cut(C, elem_size(dtype), std::max(8, lanes), false);
  RmsFwd a = fwd_args(x, residual, weight, sum_out, q, rows, C, x_stride, residual_stride, eps, cut);
  a.scales = scales;
  a.block_lanes = lanes;
  a.nblocks = by_row ? 1 : (int)ceil_div(C, block);
  a.qtype = q_dtype;
  a.q_most = q_dtype == GNNHWC_F8E4M3 ? 448.0f : 127.0f;
  return launch_fwd(a, cut, dtype, weight ? param_dtype : dtype, true, (hipStream_t)stream, "gnnhwc_rms_fwd_quant");
}

size_t gnnhwc_rms_bwd_workspace_bytes(int64_t rows, int64_t C, int dtype) {
  if (check_rows(rows, C, dtype, dtype)) return 0;
  const RowCut cut = rms_cut(C, elem_size(dtype), 8, false);
  return 256 + (size_t)rms_bwd_blocks(rows, cut) * (size_t)C * (dtype == GN_F64 ? 8 : 4);
}

int gnnhwc_rms_bwd(const void *dy, const void *ds, const void *s, const void *weight, void *dx, void *dweight, int64_t rows, int64_t C,
                   int64_t dy_stride, int64_t ds_stride, int64_t s_stride, double eps, int dtype, int param_dtype, void *workspace,
                   size_t workspace_bytes, void *stream) {
  if (const int rc = check_rows(rows, C, dtype, weight || dweight ? param_dtype : dtype)) return rc;
  if (const int rc = check_eps(eps)) return rc;
  if (rows > 0 && (!dy || !s)) return invalid("null tensor");
  if (!dx && !dweight) return GNNHWC_OK;
  if (dweight && (!workspace || ((uintptr_t)workspace & 7) || workspace_bytes < gnnhwc_rms_bwd_workspace_bytes(rows, C, dtype)))
    return fail(GNNHWC_ERR_WORKSPACE, "workspace null, misaligned or smaller than gnnhwc_rms_bwd_workspace_bytes");
  const RowCut cut = rms_cut(C, elem_size(dtype), 8, false);
  RmsBwd a = {};
  a.dy = dy; a.ds = ds; a.s = s; a.w = weight;
  a.dx = dx; a.part = dweight ? workspace : nullptr;
  a.rows = rows; a.dy_stride = dy_stride; a.ds_stride = ds_stride; a.s_stride = s_stride;
  a.eps = eps; a.inv_c = 1.0 / (double)C;
  a.C = (int)C; a.nvec = cut.nvec; a.lpr = cut.lpr; a.lpr_log2 = cut.lpr_log2;
  const int pt = weight || dweight ? param_dtype : dtype, blocks = rms_bwd_blocks(rows, cut);
  if (rows == 0 && !dweight) return GNNHWC_OK;
#define GN_CALL(S) launch_rms_bwd_##S(a, cut, pt, blocks, dweight, (hipStream_t)stream)
  return launched(GN_BY_TYPE(dtype, GN_CALL), "gnnhwc_rms_bwd");
#undef GN_CALL
}

int gnnhwc_rotary(const gnnhwc_rotary_call *c, void *stream) {
  RotaryPlan p;
  if (const int rc = plan_rotary(c, false, p)) return rc;
  if (p.empty) return GNNHWC_OK;
  const bool norm = c->q_weight != nullptr;
#define GN_CALL(S) launch_rotary_##S(p.a, p.cut, norm, (int)c->param_dtype, (hipStream_t)stream)
  return launched(GN_BY_TYPE(c->dtype, GN_CALL), "gnnhwc_rotary");
#undef GN_CALL
}

size_t gnnhwc_rotary_bwd_workspace_bytes(const gnnhwc_rotary_call *c) {
  RotaryPlan p;
  if (plan_rotary(c, true, p)) return 0;
  return 256 + (size_t)partial_bytes(p, c->dtype);
}

int gnnhwc_rotary_bwd(const gnnhwc_rotary_call *c, void *workspace, size_t workspace_bytes, void *stream) {
  RotaryPlan p;
  if (const int rc = plan_rotary(c, true, p)) return rc;
  const bool norm = c->q_weight != nullptr;
  if (p.empty && !norm) return GNNHWC_OK;
  if (!norm) {
#define GN_CALL(S) launch_rotary_##S(p.a, p.cut, false, (int)c->dtype, (hipStream_t)stream)
    return launched(GN_BY_TYPE(c->dtype, GN_CALL), "gnnhwc_rotary_bwd");
#undef GN_CALL
  }
  if (!workspace || ((uintptr_t)workspace & 7) || workspace_bytes < 256 + (size_t)partial_bytes(p, c->dtype))
    return fail(GNNHWC_ERR_WORKSPACE, "workspace null, misaligned or smaller than gnnhwc_rotary_bwd_workspace_bytes");
  p.a.part = workspace;
  void *const dw[2] = {c->q_dweight, c->kv_heads ? c->k_dweight : nullptr};
#define GN_CALL(S) launch_rotary_norm_bwd_##S(p.a, p.cut, (int)c->param_dtype, p.blocks, dw, (hipStream_t)stream)
  return launched(GN_BY_TYPE(c->dtype, GN_CALL), "gnnhwc_rotary_bwd");
#undef GN_CALL
}

size_t gnnhwc_clip_workspace_bytes(int64_t count) {
  if (count < 0) {
    invalid("negative count");
    return 0;
  }
  // (sums of more tables than these are added up on the way)
  return (size_t)(std::min<int64_t>(ceil_div(count, kClipEntries), kClipTables) * kClipBlocks + 1) * sizeof(double);
}

int gnnhwc_clip(const void *const *in, void *const *out, const int64_t *n, const int *dtype, const int *out_dtype, int64_t count,
                double max_norm, double eps, double grad_scale, void *total, int total_dtype, void *workspace, size_t workspace_bytes,
                void *stream) try {
  if (count < 0 || (count > 0 && (!in || !n || !dtype || (out && !out_dtype)))) return invalid("null array or negative count");
  if (!(max_norm >= 0)) return invalid("max_norm must not be negative");
  if (const int rc = check_eps(eps)) return rc;
  if (!(fabs(grad_scale) < INFINITY)) return invalid("grad_scale must be finite");
  if (!total) return invalid("null total");
  if (total_dtype != GN_F32 && total_dtype != GN_F64) return invalid("total must be f32 or f64");
  if (!workspace || ((uintptr_t)workspace & 7) || workspace_bytes < gnnhwc_clip_workspace_bytes(count))
    return fail(GNNHWC_ERR_WORKSPACE, "workspace null, misaligned or smaller than gnnhwc_clip_workspace_bytes");
  struct Range {
    uintptr_t from, to;
    int64_t i;
    bool written;
  };
  const bool scales = out || grad_scale != 1.0 || max_norm < INFINITY;
  std::vector<ClipEntry> list;
  std::vector<Range> ranges;
  list.reserve((size_t)count);
  if (scales) ranges.reserve((size_t)(out ? 2 * count : count));
  for (int64_t i = 0; i < count; ++i) {
    const int es = elem_size(dtype[i]), os = out ? elem_size(out_dtype[i]) : es;
    if (!es || !os) return fail(GNNHWC_ERR_INVALID_ARGUMENT, "tensor %lld: unknown dtype code", (long long)i);
    if (n[i] < 0 || n[i] > ((int64_t)1 << 42)) return fail(GNNHWC_ERR_INVALID_ARGUMENT, "tensor %lld: size out of range", (long long)i);
    if (n[i] == 0) continue;
    if (!in[i] || (out && !out[i])) return fail(GNNHWC_ERR_INVALID_ARGUMENT, "tensor %lld: null", (long long)i);
    ClipEntry e = {in[i], out ? out[i] : const_cast<void *>(in[i]), n[i], 0, dtype[i] | (out ? out_dtype[i] : dtype[i]) << 8};
    const uintptr_t a = (uintptr_t)e.in, b = (uintptr_t)e.out;
    if (scales) {
      const bool same = a == b && es == os;
      ranges.push_back({b, b + (uintptr_t)n[i] * os, i, true});
      if (!same) ranges.push_back({a, a + (uintptr_t)n[i] * es, i, false});
    }
    // neighbours in memory are one tensor (the gradients of a bucket)
    if (!list.empty()) {
      ClipEntry &l = list.back();
      if (l.types == e.types && (uintptr_t)l.in + (uintptr_t)l.n * es == a && (uintptr_t)l.out + (uintptr_t)l.n * os == b) {
        l.n += e.n;
        continue;
      }
    }
    list.push_back(e);
  }
  std::sort(ranges.begin(), ranges.end(), [](const Range &a, const Range &b) { return a.from < b.from; });
  // against the furthest end so far of what is written, and of everything
  uintptr_t any_to = 0, written_to = 0;
  for (const Range &r : ranges) {
    if (r.from < written_to || (r.written && r.from < any_to))
      return fail(GNNHWC_ERR_INVALID_ARGUMENT, "tensor %lld overlaps another one that is written", (long long)r.i);
    any_to = std::max(any_to, r.to);
    if (r.written) written_to = std::max(written_to, r.to);
  }

  int64_t chunks = 0;
  for (const ClipEntry &e : list) chunks += ceil_div(e.n, kClipChunk);
  if (chunks > 0x7fffffff) return invalid("more gradients than one call takes");
  double *part = (double *)workspace;
  ClipFinish f = {};
  f.part = part;
  f.max_norm = max_norm; f.eps = eps; f.grad_scale = grad_scale;
  f.total = total; f.total_dtype = total_dtype;
  f.in_place = !out;
  // tables of up to kClipEntries tensors, each with a launch of its own
  int64_t bytes = 0;
  auto table_at = [&](size_t first, ClipTable &t) {
    t.count = (int)std::min<size_t>(list.size() - first, kClipEntries);
    t.chunks = 0;
    for (int i = 0; i < t.count; ++i) {
      t.e[i] = list[first + (size_t)i];
      t.e[i].first_chunk = t.chunks;
      t.chunks += (unsigned)ceil_div(t.e[i].n, kClipChunk);
    }
  };
  ClipTable t;
  for (size_t at = 0; at < list.size(); at += kClipEntries) {
    table_at(at, t);
    for (int i = 0; i < t.count; ++i) bytes += t.e[i].n * elem_size(t.e[i].types & 0xff);
    const int blocks = (int)std::min<int64_t>(t.chunks, kClipBlocks);
    if (f.parts + blocks > kClipTables * kClipBlocks + 1) {
      if (const hipError_t e = launch_clip_sum(part, f.parts, (hipStream_t)stream)) return launched(e, "gnnhwc_clip");
      f.parts = 1;
    }
    if (const hipError_t e = launch_clip_norm(t, part + f.parts, blocks, (hipStream_t)stream)) return launched(e, "gnnhwc_clip");
    f.parts += blocks;
  }
  if (!scales || list.empty()) {
    t.count = 0;
    t.chunks = 0;
    return launched(launch_clip_apply(t, f, false, 1, (hipStream_t)stream), "gnnhwc_clip");
  }
  for (size_t at = 0; at < list.size(); at += kClipEntries) {
    if (list.size() > kClipEntries) table_at(at, t);
    const int blocks = (int)std::min<int64_t>(t.chunks, 2 * kClipBlocks);
    if (const hipError_t e = launch_clip_apply(t, f, bytes > kCachedBytes, blocks, (hipStream_t)stream)) return launched(e, "gnnhwc_clip");
    f.total = nullptr;  // written by the first launch
  }
  return GNNHWC_OK;
} catch (...) {
  return fail(GNNHWC_ERR_LAUNCH, "gnnhwc_clip: out of host memory");
}

}  // extern "C"
