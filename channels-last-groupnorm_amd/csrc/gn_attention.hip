// C ABI of the attention (declared in include/gnnhwc_tokens.h): argument checks and launch planning.
#include <hip/hip_runtime.h>
#include <math.h>

#include <algorithm>

#include "gn_error.h"
#include "gn_window_args.h"

namespace gn {
namespace {

constexpr int64_t kMostTokens = (int64_t)1 << 30;
constexpr int64_t kFineKeys = 64;  // (where 64 are seen, 1.44 without)
constexpr int64_t kMostItems = ((int64_t)1 << 23) - 64;  // workgroups of up to 512 threads: a launch has fewer than 2^32

int invalid(const char *what) { return fail(GNNHWC_ERR_INVALID_ARGUMENT, "%s", what); }
int launched(hipError_t e, const char *what) {
  return e == hipSuccess ? GNNHWC_OK : fail(GNNHWC_ERR_LAUNCH, "%s: %s", what, hipGetErrorString(e));
}
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
size_t round_up(size_t n) { return (n + 255) / 256 * 256; }

int put_rows(HeadRows &r, const void *base, const int64_t (&stride)[3], int64_t batch, int64_t tokens, int64_t heads, int64_t es, const char *name) {
  r = {};
  if (batch == 0 || tokens == 0) return GNNHWC_OK;
  if (!base) return fail(GNNHWC_ERR_INVALID_ARGUMENT, "%s is null", name);
  const int64_t size[3] = {batch, tokens, heads};
  int64_t bytes[3];
  for (int i = 0; i < 3; ++i) {
    const int64_t s = size[i] == 1 ? 0 : stride[i];
    if (s < 0 || s > ((int64_t)1 << 56) / size[i]) return fail(GNNHWC_ERR_INVALID_ARGUMENT, "%s: stride out of range", name);
    bytes[i] = s * es;
    if (bytes[i] % 16) return fail(GNNHWC_ERR_INVALID_ARGUMENT, "%s: its strides must be whole multiples of 16 bytes", name);
  }
  if ((uintptr_t)base % 16) return fail(GNNHWC_ERR_INVALID_ARGUMENT, "%s must be aligned to 16 bytes", name);
  if (bytes[1] >= (int64_t)1 << 25) return fail(GNNHWC_ERR_INVALID_ARGUMENT, "%s: a token's stride must be below 2^25 bytes", name);
  r.base = base;
  r.batch_bytes = bytes[0];
  r.token_bytes = (int)bytes[1];
  r.head_bytes = bytes[2];
  return GNNHWC_OK;
}

// The order in which the workgroups' work goes to the dies, and what they divide by to find theirs: once all else of a is set.
void put_order(WindowArgs &a) {
  const int heads = a.B * a.K;
  a.per_head = heads ? a.items / heads : 0;
  a.order = heads % 8 == 0 ? kHeadsInTurn : a.lengths ? kInTurn : kStretches;
  a.by_group = make_divisor(std::max(1, a.group), 0);
  a.by_splits = make_divisor(std::max(1, a.splits), 0);
  a.by_tiles = make_divisor(std::max(1, a.tiles), 0);
  a.by_K = make_divisor(std::max(1, a.K), 0);
  a.by_shares = make_divisor(std::max(1, a.shares), 0);
  a.by_sink_parts = make_divisor(std::max(1, a.sink_parts), 0);
  a.by_sink_sets = make_divisor(std::max(1, a.sink_sets), 0);
  a.by_per_head = make_divisor(std::max(1, a.per_head), 0);
  a.by_L = make_divisor(std::max(1, a.L), 0);
  a.by_H = make_divisor(std::max(1, a.H), 0);
}

struct WindowPlan {
  WindowArgs a, kv, sinks;  // queries' tiles, keys' tiles, sinks
  bool empty, few;          // few: 32 rows of a key head at a time, see window_few_kernel
  size_t delta, largest, part_q, part_k, part_v, bytes;  // the workspace (forward: part_k references and sums, part_v rows)
};

// Workgroups that share the work of each of `items`, of `steps` steps: a CU takes `thick` of them at once in the time of one, each
// has some steps' time of its own, and what they leave has to be joined.  (training of 1500 tokens, 8 heads over 2 of 128, causal, in
// bfloat16: 99 us, unshared 294; of a padded float32 batch, 3 x 1961, 6 over 2 of 40: 250 and 500)
// mean: steps of an item on average; where they are uneven, the CUs are as good as evenly loaded, but the longest item has to end, too.
// (float32, 4 x 800 tokens, 8 heads over 2 of 96, causal: forward 94 us unshared, 78 by two; dk and dv 383 by four, 313 by eight)
int64_t shares_of(int64_t items, int64_t steps, int64_t mean, int64_t thick, int64_t most) {
  if (items == 0) return 1;
  // (in steps of which a CU takes `thick` at once: 1.7 us for float32, 0.5 for 16 bits, where the second launch is 4 us and a share's
  // rows, written and read, 13 ns)
  const int64_t join = thick == 1 ? 3 : 8, rows = thick == 1 ? 128 : 32, overhead = thick == 1 ? 1 : 3;
  auto cost = [&](int64_t s) {
    const int64_t joined = s > 1 ? join + items * s / rows : 0;
    if (mean < steps) return std::max(items * (mean + overhead * s) / kNumCU, thick * (ceil_div(steps, s) + overhead)) + joined;
    return std::max(ceil_div(items * s, kNumCU), thick) * (ceil_div(steps, s) + overhead) + joined;
  };
  int64_t best = 1;
  for (int64_t s = 2; s <= most && s <= steps / 2; ++s)
    if (cost(s) < cost(best)) best = s;
  return best;
}

int plan_window(const gnnhwc_window_call *c, bool backward, WindowPlan &p) {
  if (!c) return invalid("null call");
  const int64_t es = c->dtype == GN_F32 ? 4 : c->dtype == GN_F16 || c->dtype == GN_BF16 ? 2 : 0;
  if (!es) return fail(GNNHWC_ERR_INVALID_ARGUMENT, "dtype code %lld: attention takes f32, f16 or bf16", (long long)c->dtype);
  if (c->batch < 0 || c->tokens < 0 || c->keys < 0) return invalid("batch, tokens and keys must not be negative");
  if (c->tokens > kMostTokens || c->keys > kMostTokens || c->batch > kMostTokens) return invalid("batch, tokens or keys out of range: at most 2^30");
  if (c->heads < 1 || c->kv_heads < 1 || c->heads > 65535 || c->heads % c->kv_heads) return invalid("heads must be 1 to 65535 and a multiple of kv_heads");
  if (c->head_dim < 8 || c->head_dim > 256 || c->head_dim % 8) return invalid("head_dim must be a multiple of 8 from 8 to 256");
  if (es == 4 && c->head_dim > 128) return invalid("head_dim must be 128 or less in f32");
  if (c->window < -1 || c->sinks < 0) return invalid("window must be -1 or more, and sinks not negative");
  if (c->length_type != 0 && c->length_type != 1) return invalid("length_type must be 0 (int32) or 1 (int64)");
  if (!(c->scale > 0 && c->scale < INFINITY)) return invalid("scale must be positive and finite");
  if (!c->at_end && c->tokens > c->keys) return invalid("more queries than keys: the queries are the last of the keys' tokens");
  if (backward && c->at_end) return invalid("attention against a cache has no backward");
  p = {};
  WindowArgs &a = p.a;
  const int64_t rows = c->heads, kv = c->kv_heads;
  if (const int rc = put_rows(a.q, c->q, c->q_stride, c->batch, c->tokens, rows, es, "q")) return rc;
  if (const int rc = put_rows(a.k, c->k, c->k_stride, c->batch, c->keys, kv, es, "k")) return rc;
  if (const int rc = put_rows(a.v, c->v, c->v_stride, c->batch, c->keys, kv, es, "v")) return rc;
  if (const int rc = put_rows(a.out, c->out, c->out_stride, c->batch, c->tokens, rows, es, "out")) return rc;
  if (backward) {
    if (const int rc = put_rows(a.dout, c->out_grad, c->out_grad_stride, c->batch, c->tokens, rows, es, "out_grad")) return rc;
    if (const int rc = put_rows(a.dq, c->q_grad, c->q_grad_stride, c->batch, c->tokens, rows, es, "q_grad")) return rc;
    if (const int rc = put_rows(a.dk, c->k_grad, c->k_grad_stride, c->batch, c->keys, kv, es, "k_grad")) return rc;
    if (const int rc = put_rows(a.dv, c->v_grad, c->v_grad_stride, c->batch, c->keys, kv, es, "v_grad")) return rc;
    if (c->batch && c->tokens && !c->lse) return invalid("lse is null");
  }
  if ((uintptr_t)c->out_rest % 16) return invalid("out_rest must be 16-byte aligned");
  a.rest = es == 2 ? c->out_rest : nullptr;
  a.lse = c->lse;
  a.lengths = c->lengths;
  a.length_type = (int)c->length_type;
  a.at_end = c->at_end != 0;
  a.B = (int)c->batch; a.L = (int)c->tokens; a.S = (int)c->keys; a.H = (int)c->heads; a.K = (int)c->kv_heads; a.D = (int)c->head_dim;
  a.group = a.H / a.K;
  a.causal = c->causal != 0;
  a.left = (int)(c->window < 0 ? kMostTokens : std::min(c->window, kMostTokens));
  a.right = a.causal ? 0 : a.left;
  a.sinks = c->window < 0 ? 0 : (int)std::min(c->sinks, kMostTokens);  // (without a bound all are seen)
  a.scale = (float)c->scale;
  a.scale_log2 = (float)(c->scale * 1.4426950408889634);
  if (!(a.scale > 0 && a.scale_log2 < INFINITY)) return invalid("scale must be positive and finite");
  if (a.sinks >= a.S || (a.left >= a.S - 1 && a.right >= (a.causal ? 0 : a.S - 1))) {  // all see all
    a.left = kMostTokens;
    a.right = a.causal ? 0 : a.left;
    a.sinks = 0;
  }
  // Rounding the weights of the second product leaves the forward's result inexact by more than its own rounding where they are few,
  // and the gradients, which are small differences there, by half as much again: two tokens of 64 channels in bfloat16 1.58 times
  // what rounding dq alone leaves, 1.41 with the weights and what rounding them left.
  a.fine = es == 2 && std::min<int64_t>(a.S, (int64_t)a.left + a.right + 1 + a.sinks) <= kFineKeys;
  a.tiles = (int)ceil_div(a.L, kQueries);
  a.splits = a.shares = 1;
  const int64_t items = (int64_t)a.tiles * a.H * a.B, lse = (int64_t)a.B * a.H * a.L;
  if (items > kMostItems || (int64_t)a.H * a.B > kMostItems) return invalid("too many tokens and heads for one call");
  a.items = (int)items;
  p.empty = items == 0;
  const int64_t width = window_width(a.D), step = es == 2 ? 64 : 32;  // tokens of the other side that a step takes
  // workgroups that a CU takes at once: as many as hide each other's latencies (float32 is bound by its products)
  const int64_t thick = es == 4 ? 1 : width <= 64 ? 3 : width <= 128 ? 2 : 1;
  const int64_t reach = (int64_t)a.left + a.right + kQueries;
  const int64_t keys = ceil_div(std::min<int64_t>(a.S, reach + a.sinks), step), queries = ceil_div(std::min<int64_t>(a.L, reach), step) * a.group;
  // of a causal walk the first tiles see less: the mean over p of min(p, n) keys, n being the most that one sees
  const int64_t seen = std::min<int64_t>(a.S, reach), lacking = a.causal ? seen * seen / (2 * std::max<int64_t>(1, a.S)) : 0;
  const int64_t mean_keys = a.L < a.S ? keys : std::max<int64_t>(1, keys - lacking / step);
  p.bytes = GNNHWC_WINDOW_NO_WORKSPACE;
  if (!backward) {
    const int64_t few_rows = (int64_t)a.L * a.group;
    // The kernel for few queries has tiles of 32 rows, all of a workgroup's wavefronts share a tile's keys, and its queries are
    // read by nobody else; the other has 128 rows, a wavefront's 32 to itself, and reads keys once for all.  The first is faster
    // while its tiles leave CUs without work (wide heads have fewer wavefronts): bfloat16, 8 samples of 8 heads of 64, 100 queries,
    // 2000 keys 14.5 us against 22.2, one of 20 heads of 64, 200 tokens 6.0 against 9.3; 4 samples of 8 heads of 128, 250 queries,
    // 2000 keys 29.7 against 28.9.  float32 is bound by its products, which the first shares evenly: what counts are the tiles of keys
    // that all its tiles of rows visit.  2 samples of 12 heads of 64, 200 queries, window 50 (840 of them) 8.6 us against 20.3, 4
    // of 8 heads, 250 queries, 2000 keys (16000) 60.6 against 52.6; heads of 128: 840 23.1 against 47.1, 980 36.9 against 30.3.
    // (16 samples of 16 heads of 128, 1000 keys: 32 queries 19.3 against 25.1, 64 queries 33.6 against 26.4)
    const int64_t few_tiles = (int64_t)a.B * a.K * ceil_div(few_rows, 32);
    const int64_t visits = few_tiles * ceil_div(std::min<int64_t>(a.S, (int64_t)a.left + a.right + a.sinks + 32 / std::min(a.group, 32) + 32), 32);
    if (es == 2) p.few = few_tiles <= (width <= 64 ? kNumCU : kNumCU * 3 / 4);
    else p.few = few_tiles <= 2 * kNumCU && visits <= (width <= 64 ? 8192 : 900);
    p.few |= few_rows <= 32;
    if (p.empty) return GNNHWC_OK;
    if (p.few) {
      a.tiles = (int)ceil_div(few_rows, 32);
      const int64_t heads = (int64_t)a.B * a.K * a.tiles;
      // Keys that a tile's rows see at most, in tiles of 32 and of a wavefront one takes 1.5 us of waiting for it (float32: 3, of its
      // products), until the memory is what is waited for; a workgroup has 2 us besides, and joining takes a second launch of 4.  (one
      // token of 8 heads of 128 against 2000: one workgroup a head 18 us, two 15.5, five 12.2, nine, as here, 11.1; 8 heads of 64
      // against 300: one, as here, 6.2, three 8.2; in float32 one 14.6, three, as here, 10.8)
      const int64_t tiles = ceil_div(std::min<int64_t>(a.S, (int64_t)a.left + a.right + a.L + a.sinks + 64), 32), waves = few_waves((int)width, (int)es);
      const int64_t each = es == 4 ? 6 : 3;
      auto cost = [&](int64_t s) { return ceil_div(heads * s, kNumCU) * (4 + each * ceil_div(tiles, s * waves)) + (s > 1 ? 8 : 0); };
      for (int64_t s = 2; s <= 64 && s <= tiles; ++s)
        if (cost(s) < cost(a.splits)) a.splits = (int)s;
      a.items = (int)(heads * a.splits);
    } else {
      a.splits = (int)shares_of(items, keys, mean_keys, thick, 16);
      a.items = (int)(items * a.splits);
    }
    put_order(a);
    if (a.splits > 1) {
      p.part_v = round_up((size_t)a.splits * lse * 2 * sizeof(float));
      p.bytes += p.part_v + (size_t)a.splits * lse * a.D * sizeof(float);
    }
    return GNNHWC_OK;
  }
  p.kv = p.sinks = a;
  if (items) {
    a.splits = (int)shares_of(items, keys, mean_keys, thick, 16);
    a.items = (int)(items * a.splits);
  }
  put_order(a);
  WindowArgs &w = p.kv, &k = p.sinks;
  w.tiles = (int)ceil_div(a.S, kQueries);
  const int64_t heads = (int64_t)a.B * a.K, tiles = heads * w.tiles;
  // (of 16 bits, where the joins weigh more, by the longest alone: 4500 tokens, 16 heads over 4 of 128, 679 us so, 711 by the mean)
  const int64_t mean_queries = es == 2 || a.L < a.S ? queries : std::max<int64_t>(1, queries - lacking / step * a.group);
  w.shares = (int)shares_of(tiles, queries, mean_queries, es == 4 ? 1 : width <= 64 ? 2 : 1, 32);
  if (tiles * w.shares > kMostItems) return invalid("too many tokens and heads for one call");
  w.items = (int)(tiles * w.shares);
  k.items = w.sink_sets = w.sink_parts = 0;
  if (w.sinks > 0 && w.items > 0) {
    const int waves = few_waves((int)width, (int)es);
    w.sink_sets = (int)ceil_div(w.sinks, 32);
    const int64_t sets = heads * w.sink_sets, steps = ceil_div(a.L, 32) * a.group;
    // as many workgroups as there are CUs, down to one step a wavefront (float32, 6 sets of 186 steps: 11 shares 28.7 us, 43 16.3)
    const int64_t sink_shares = std::clamp<int64_t>(kNumCU / std::max<int64_t>(1, sets), 1, std::max<int64_t>(1, steps / waves));
    // (rows are added up by 256 threads or fewer each)
    if (sets * sink_shares > kMostItems || heads * w.sinks / std::max(1, 64 / a.D) > 2 * kMostItems) return invalid("too many tokens and heads for one call");
    w.sink_parts = (int)sink_shares;
    k = w;
    k.items = (int)(sets * sink_shares);
    put_order(k);
  }
  put_order(w);
  const size_t floats = round_up((size_t)lse * sizeof(float));
  const size_t part = round_up(((size_t)heads * w.sink_sets * w.sink_parts * 32 + (w.shares > 1 ? (size_t)tiles * w.shares * kQueries : 0)) * a.D * sizeof(float));
  p.delta = 0;
  p.largest = floats;
  p.part_q = p.largest + (c->dtype == GN_F16 ? floats : 0);
  p.part_k = p.part_q + (a.splits > 1 ? round_up((size_t)a.splits * lse * a.D * sizeof(float)) : 0);
  p.part_v = p.part_k + part;
  p.bytes += p.part_v + part;
  return GNNHWC_OK;
}

#define GN_BY_TYPE(dtype, call) ((dtype) == GN_F32 ? call(f32) : (dtype) == GN_F16 ? call(f16) : call(bf16))

}  // namespace
}  // namespace gn

using namespace gn;

extern "C" {

size_t gnnhwc_window_workspace_bytes(const gnnhwc_window_call *c) {
  WindowPlan p;
  if (plan_window(c, false, p)) return 0;
  return p.bytes;
}

int gnnhwc_window(const gnnhwc_window_call *c, void *workspace, size_t workspace_bytes, void *stream) {
  WindowPlan p;
  if (const int rc = plan_window(c, false, p)) return rc;
  if (p.bytes > GNNHWC_WINDOW_NO_WORKSPACE && (!workspace || (uintptr_t)workspace % GNNHWC_WINDOW_WORKSPACE_ALIGNMENT || workspace_bytes < p.bytes))
    return fail(GNNHWC_ERR_WORKSPACE, "workspace null, misaligned or smaller than gnnhwc_window_workspace_bytes");
  if (p.empty) return GNNHWC_OK;
  p.a.part_k = (float *)workspace;
  p.a.part_v = (float *)((char *)workspace + p.part_v);
#define GN_CALL(S) launch_window_forward_##S(p.a, p.few, (hipStream_t)stream)
  return launched(GN_BY_TYPE(c->dtype, GN_CALL), "gnnhwc_window");
#undef GN_CALL
}

size_t gnnhwc_window_bwd_workspace_bytes(const gnnhwc_window_call *c) {
  WindowPlan p;
  if (plan_window(c, true, p)) return 0;
  return p.bytes;
}

int gnnhwc_window_bwd(const gnnhwc_window_call *c, void *workspace, size_t workspace_bytes, void *stream) {
  WindowPlan p;
  if (const int rc = plan_window(c, true, p)) return rc;
  if (!workspace || (uintptr_t)workspace % GNNHWC_WINDOW_WORKSPACE_ALIGNMENT || workspace_bytes < p.bytes)
    return fail(GNNHWC_ERR_WORKSPACE, "workspace null, misaligned or smaller than gnnhwc_window_bwd_workspace_bytes");
  for (WindowArgs *a : {&p.a, &p.kv, &p.sinks}) {
    a->delta = (float *)((char *)workspace + p.delta);
    a->largest = (float *)((char *)workspace + p.largest);
    a->part_q = (float *)((char *)workspace + p.part_q);
    a->part_k = (float *)((char *)workspace + p.part_k);
    a->part_v = (float *)((char *)workspace + p.part_v);
  }
  if (p.kv.items == 0) return GNNHWC_OK;  // (then there are no queries either)
#define GN_CALL(S) launch_window_backward_##S(p.a, p.kv, p.sinks, (hipStream_t)stream)
  return launched(GN_BY_TYPE(c->dtype, GN_CALL), "gnnhwc_window_bwd");
#undef GN_CALL
}

}  // extern "C"
