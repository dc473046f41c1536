// Eager calls of the operators for token streams without Python on the way (see gn_torch.cpp): checks, allocations, the C ABI
// call and the autograd node.  Each takes ordinary calls only and answers NotImplemented to everything else, errors included;
// the caller then runs the general implementation behind the gnop:: operators.
#include "gn_torch.h"

#include <cmath>
#include <vector>

#include <ATen/hip/EmptyTensor.h>
#include <torch/csrc/autograd/variable.h>

#include "../../include/gnnhwc_tokens.h"

namespace {

using namespace gn_torch;

// The C ABI's entry points, handed over by address as in gn_torch.cpp.
struct Entry {
  decltype(&gnnhwc_last_error) last_error;
  decltype(&gnnhwc_rms_fwd) rms_fwd;
  decltype(&gnnhwc_rms_fwd_quant) rms_fwd_quant;
  decltype(&gnnhwc_rms_bwd_workspace_bytes) rms_bwd_workspace_bytes;
  decltype(&gnnhwc_rms_bwd) rms_bwd;
  decltype(&gnnhwc_rotary) rotary;
  decltype(&gnnhwc_rotary_bwd_workspace_bytes) rotary_bwd_workspace_bytes;
  decltype(&gnnhwc_rotary_bwd) rotary_bwd;
  decltype(&gnnhwc_clip_workspace_bytes) clip_workspace_bytes;
  decltype(&gnnhwc_clip) clip;
  decltype(&gnnhwc_window_workspace_bytes) window_workspace_bytes;
  decltype(&gnnhwc_window) window;
  decltype(&gnnhwc_window_bwd_workspace_bytes) window_bwd_workspace_bytes;
  decltype(&gnnhwc_window_bwd) window_bwd;
  decltype(&gnnhwc_dropout) dropout;
} abi = {};

void check(int rc, const char *what) { TORCH_CHECK(rc == 0, what, " failed (code ", rc, "): ", abi.last_error()); }
// Memory on like's device from the caching allocator, without the dispatcher: small calls are bound by the host.
Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const Tensor &like) {
  return Tensor(at::detail::empty_cuda(sizes, type, like.device(), std::nullopt));
}
Tensor workspace(size_t bytes, const Tensor &like, const char *what) {
  TORCH_CHECK(bytes != 0, what, ": ", abi.last_error());
  return fresh({(int64_t)bytes}, at::kByte, like);
}
PyObject *decline() { Py_RETURN_NOTIMPLEMENTED; }
Tensor defined(const optional<Tensor> &t) { return t.has_value() ? *t : Tensor(); }
void *ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

// (..., C) as rows of contiguous channels with one stride from row to row.
struct Rows {
  int64_t count = 0, C = 0, stride = 0;
};
bool rows_of(const Tensor &t, Rows &r) {
  const int64_t nd = t.dim();
  if (nd < 1 || t.numel() == 0) return false;
  r.C = t.size(nd - 1);
  if (r.C != 1 && t.stride(nd - 1) != 1) return false;
  r.count = 1;
  r.stride = r.C;
  int64_t expect = 0;
  for (int64_t d = nd - 2; d >= 0; --d) {
    if (t.size(d) == 1) continue;
    if (r.count == 1) r.stride = t.stride(d);
    else if (t.stride(d) != expect) return false;
    r.count *= t.size(d);
    expect = t.stride(d) * t.size(d);
  }
  return true;
}
bool weight_fits(const Tensor &w, const Tensor &x, int64_t n) {
  return plain(w, x.device()) && w.dim() == 1 && w.numel() == n && w.is_contiguous() &&
         (w.scalar_type() == x.scalar_type() || (is_half(x.scalar_type()) && w.scalar_type() == at::kFloat));
}
bool eps_of(PyObject *o, double &eps) {
  if (!PyFloat_CheckExact(o)) return false;
  eps = PyFloat_AS_DOUBLE(o);
  return eps >= 0 && std::isfinite(eps);
}
int param_code(const Tensor &w, const Tensor &x) { return code_of(w.defined() ? w.scalar_type() : x.scalar_type()); }
PyObject *wrap_all(std::initializer_list<Tensor> ts) {
  PyObject *tuple = PyTuple_New((Py_ssize_t)ts.size());
  Py_ssize_t i = 0;
  for (const Tensor &t : ts) {
    PyObject *o = tuple ? THPVariable_Wrap(t) : nullptr;
    if (!o) {
      Py_XDECREF(tuple);
      return nullptr;
    }
    PyTuple_SET_ITEM(tuple, i++, o);
  }
  return tuple;
}

// ---- root-mean-square norm ----
struct NormCall {
  Tensor x, weight, residual;  // weight, residual: possibly undefined
  Rows xr, rr;
  double eps = 0;
};
// The arguments x, weight, eps, residual; false: not an ordinary call.
bool norm_call(PyObject *const *args, NormCall &c) {
  optional<Tensor> x, weight, residual;
  if (!tensor_or_none(args[0], x) || !x.has_value() || !ordinary_thread() || !tensor_or_none(args[1], weight) || !eps_of(args[2], c.eps) ||
      !tensor_or_none(args[3], residual))
    return false;
  c.x = *x;
  const int dt = code_of(c.x.scalar_type());
  if (dt < 0 || !plain(c.x, c.x.device()) || !rows_of(c.x, c.xr)) return false;
  c.weight = defined(weight);
  c.residual = defined(residual);
  if (c.weight.defined() && !weight_fits(c.weight, c.x, c.xr.C)) return false;
  if (c.residual.defined() && (!plain(c.residual, c.x.device()) || c.residual.scalar_type() != c.x.scalar_type() ||
                               c.residual.sizes() != c.x.sizes() || !rows_of(c.residual, c.rr)))
    return false;
  return true;
}
bool wants_grad(std::initializer_list<Tensor> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor &t : ts)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}
// (the sum is left undefined unless there is a residual and it is wanted)
void run_norm(const NormCall &c, bool want_sum, Tensor &y, Tensor &sum) {
  const c10::DeviceGuard guard(c.x.device());
  const at::AutoDispatchBelowADInplaceOrView below;
  const OperatorRange range("gnop::rms_norm");
  y = fresh(c.x.sizes(), c.x.scalar_type(), c.x);
  if (want_sum && c.residual.defined()) sum = fresh(c.x.sizes(), c.x.scalar_type(), c.x);
  check(abi.rms_fwd(c.x.data_ptr(), ptr(c.residual), ptr(c.weight), ptr(sum), y.data_ptr(), c.xr.count, c.xr.C, c.xr.stride, c.rr.stride, c.eps,
                    code_of(c.x.scalar_type()), param_code(c.weight, c.x), stream_of(c.x)),
        "gnop::rms_norm");
}

struct NormNode : public torch::autograd::Function<NormNode> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext *ctx, const Tensor &x, const optional<Tensor> &weight,
                                                const optional<Tensor> &residual, NormCall *c) {
    Tensor y, sum;
    run_norm(*c, true, y, sum);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({sum.defined() ? sum : x, weight.value_or(Tensor())});
    ctx->saved_data["eps"] = c->eps;
    ctx->saved_data["residual"] = sum.defined();
    if (!sum.defined()) return {y};
    return {y, sum};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const bool residual = ctx->saved_data["residual"].toBool();
    const double eps = ctx->saved_data["eps"].toDouble();
    const Tensor s = saved[0], weight = saved[1], dy = grads[0], ds = residual ? grads[1] : Tensor();
    if (!dy.defined()) return {ds, Tensor(), ds, Tensor()};  // only the sum was used
    Tensor dx, dw;
    Rows sr, yr, dr;
    const c10::Device device = dy.device();
    // Saved-tensor hooks may have returned anything, and gradients need not be plain: the operator takes (or refuses) those.
    if (at::GradMode::is_enabled() || !ordinary_dispatch() || !plain(dy, device) || !plain(s, device) || s.sizes() != dy.sizes() ||
        s.scalar_type() != dy.scalar_type() || !rows_of(s, sr) || !rows_of(dy, yr) || (weight.defined() && !weight_fits(weight, s, sr.C)) ||
        (ds.defined() && (!plain(ds, device) || ds.scalar_type() != s.scalar_type() || ds.sizes() != s.sizes() || !rows_of(ds, dr)))) {
      using Signature = std::tuple<Tensor, Tensor>(const Tensor &, const optional<Tensor> &, const Tensor &, const optional<Tensor> &, double);
      const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("gnop::rms_norm_bwd", "").typed<Signature>();
      std::tie(dx, dw) = op.call(dy, ds.defined() ? optional<Tensor>(ds) : std::nullopt, s,
                                 weight.defined() ? optional<Tensor>(weight) : std::nullopt, eps);
    } else {
      const c10::DeviceGuard guard(device);
      const at::AutoDispatchBelowADInplaceOrView below;
      const OperatorRange range("gnop::rms_norm_bwd");
      const int dt = code_of(s.scalar_type());
      // (edges count the inputs that are there: x, weight, residual)
      const bool wants_dx = ctx->needs_input_grad(0) || (residual && ctx->needs_input_grad(weight.defined() ? 2 : 1));
      if (wants_dx) dx = fresh(s.sizes(), s.scalar_type(), s);
      Tensor ws;
      size_t bytes = 0;
      if (weight.defined() && ctx->needs_input_grad(1)) {
        dw = fresh({sr.C}, weight.scalar_type(), weight);
        bytes = abi.rms_bwd_workspace_bytes(sr.count, sr.C, dt);
        ws = workspace(bytes, s, "gnop::rms_norm_bwd");
      }
      check(abi.rms_bwd(dy.data_ptr(), ptr(ds), s.data_ptr(), ptr(weight), ptr(dx), ptr(dw), sr.count, sr.C, yr.stride, dr.stride, sr.stride,
                        eps, dt, param_code(weight, s), ptr(ws), bytes, stream_of(s)),
            "gnop::rms_norm_bwd");
    }
    return {dx, weight.defined() ? dw : Tensor(), residual ? dx : Tensor(), Tensor()};
  }
};

// rms_norm(x, weight, eps, residual, return_sum) -> y, (y, s) or NotImplemented
PyObject *rms_norm(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  TORCH_CHECK(nargs == 5, "rms_norm takes 5 arguments");
  NormCall c;
  if (!PyBool_Check(args[4]) || !norm_call(args, c)) return decline();
  const bool return_sum = args[4] == Py_True;
  const int64_t most = c.x.scalar_type() == at::kDouble ? 8192 : 16384;
  if (c.xr.C > most || c.xr.count > 0x7fffffff) return decline();
  Tensor y, sum;
  {
    const WithoutGil released;
    if (wants_grad({c.x, c.weight, c.residual})) {
      const auto weight = c.weight.defined() ? optional<Tensor>(c.weight) : std::nullopt;
      const auto residual = c.residual.defined() ? optional<Tensor>(c.residual) : std::nullopt;
      const auto out = NormNode::apply(c.x, weight, residual, &c);
      y = out[0];
      if (out.size() > 1) sum = out[1];
    } else {
      run_norm(c, return_sum, y, sum);
    }
  }
  if (!return_sum) return THPVariable_Wrap(y);
  return wrap_all({y, c.residual.defined() ? sum : c.x});
  END_HANDLE_TH_ERRORS
}

// rms_norm_quant(x, weight, eps, residual, return_sum, out_dtype, block) -> (q, scales), (q, scales, s) or NotImplemented
PyObject *rms_norm_quant(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  TORCH_CHECK(nargs == 7, "rms_norm_quant takes 7 arguments");
  NormCall c;
  if (!PyBool_Check(args[4]) || !THPDtype_Check(args[5]) || !norm_call(args, c) || wants_grad({c.x, c.weight, c.residual})) return decline();
  const bool return_sum = args[4] == Py_True;
  const at::ScalarType out = reinterpret_cast<THPDtype *>(args[5])->scalar_type;
  if ((out != at::kFloat8_e4m3fn && out != at::kChar) || c.x.scalar_type() == at::kDouble || c.xr.C > 16384 || c.xr.count > 0x7fffffff) return decline();
  int64_t block = 0;
  if (args[6] != Py_None) {
    if (!PyLong_CheckExact(args[6])) return decline();
    block = PyLong_AsLongLong(args[6]);
    if (PyErr_Occurred()) {
      PyErr_Clear();
      return decline();
    }
    if (block < 1 || (block < c.xr.C && (block < 16 || block > 256 || (block & (block - 1))))) return decline();
  }
  Tensor q, scales, sum;
  {
    const WithoutGil released;
    const c10::DeviceGuard guard(c.x.device());
    const at::AutoDispatchBelowADInplaceOrView below;
    const OperatorRange range("gnop::rms_norm_quant");
    c10::SmallVector<int64_t, 6> shape(c.x.sizes().begin(), c.x.sizes().end());
    q = fresh(shape, out, c.x);
    shape.back() = block == 0 || block >= c.xr.C ? 1 : (c.xr.C + block - 1) / block;
    scales = fresh(shape, at::kFloat, c.x);
    if (return_sum && c.residual.defined()) sum = fresh(c.x.sizes(), c.x.scalar_type(), c.x);
    check(abi.rms_fwd_quant(c.x.data_ptr(), ptr(c.residual), ptr(c.weight), ptr(sum), q.data_ptr(), (float *)scales.data_ptr(), c.xr.count, c.xr.C,
                            c.xr.stride, c.rr.stride, block, c.eps, code_of(c.x.scalar_type()), param_code(c.weight, c.x),
                            out == at::kChar ? GNNHWC_I8 : GNNHWC_F8E4M3, stream_of(c.x)),
          "gnop::rms_norm_quant");
  }
  if (!return_sum) return wrap_all({q, scales});
  return wrap_all({q, scales, c.residual.defined() ? sum : c.x});
  END_HANDLE_TH_ERRORS
}

// ---- rotary positions ----
struct RotaryArgs {
  Tensor positions, frequencies;
  std::vector<int64_t> sections;
  bool interleaved = false;
  double eps = 0;
};
// Whether positions and frequencies go with q; fills the call but for tensors and weights.
bool rotary_call(const Tensor &q, const Tensor &k, const RotaryArgs &a, gnnhwc_rotary_call &c) {
  const int64_t axes = (int64_t)a.sections.size(), B = q.size(0), L = q.size(1);
  if (axes < 1 || axes > 4) return false;
  c.batch = B;
  c.tokens = L;
  c.heads = q.size(2);
  c.kv_heads = k.defined() ? k.size(2) : 0;
  c.head_dim = q.size(3);
  c.axes = axes;
  int64_t end = 0;
  for (int64_t i = 0; i < axes; ++i) {
    if (a.sections[i] < 0) return false;
    end += a.sections[i];
    c.section_end[i] = end;
  }
  const Tensor &f = a.frequencies, &p = a.positions;
  if (!plain(f, q.device()) || f.scalar_type() != at::kFloat || f.dim() != 1 || f.numel() != end || !f.is_contiguous()) return false;
  if (!plain(p, q.device())) return false;
  switch (p.scalar_type()) {
    case at::kInt: c.position_type = 0; break;
    case at::kLong: c.position_type = 1; break;
    case at::kFloat: c.position_type = 2; break;
    default: return false;
  }
  const int64_t nd = p.dim();
  if (nd == 3 || (nd == 2 && !(axes == 1 && p.size(1) == L))) {  // (B or 1, L, axes) or (L, axes)
    if (p.size(nd - 1) != axes || p.size(nd - 2) != L || (axes > 1 && p.stride(nd - 1) != 1)) return false;
    if (nd == 3 && p.size(0) != 1 && p.size(0) != B) return false;
    c.position_stride[0] = nd == 3 && p.size(0) != 1 ? p.stride(0) : 0;
    c.position_stride[1] = p.stride(nd - 2);
  } else if (axes == 1 && (nd == 1 || nd == 2)) {  // (L,) or (B or 1, L)
    if (p.size(nd - 1) != L || (nd == 2 && p.size(0) != 1 && p.size(0) != B)) return false;
    c.position_stride[0] = nd == 2 && p.size(0) != 1 ? p.stride(0) : 0;
    c.position_stride[1] = p.stride(nd - 1);
  } else {
    return false;
  }
  c.interleaved = a.interleaved;
  c.positions = p.data_ptr();
  c.frequencies = (const float *)f.data_ptr();
  c.eps = a.eps;
  c.dtype = c.param_dtype = code_of(q.scalar_type());
  return true;
}
void put_strides(const Tensor &t, int64_t (&s)[3]) {
  for (int i = 0; i < 3; ++i) s[i] = t.stride(i);
}
bool heads_fit(const Tensor &t, const c10::Device &device) {
  return plain(t, device) && t.dim() == 4 && t.numel() > 0 && (t.stride(3) == 1 || t.size(3) == 1);
}
bool like_q(const Tensor &k, const Tensor &q) {
  return heads_fit(k, q.device()) && k.scalar_type() == q.scalar_type() && k.size(0) == q.size(0) && k.size(1) == q.size(1) && k.size(3) == q.size(3);
}
bool put_weights(const Tensor &qw, const Tensor &kw, const Tensor &q, bool has_k, gnnhwc_rotary_call &c) {
  if (has_k ? qw.defined() != kw.defined() : kw.defined()) return false;
  if (!qw.defined()) return true;
  if (!weight_fits(qw, q, c.head_dim) || (has_k && (!weight_fits(kw, q, c.head_dim) || kw.scalar_type() != qw.scalar_type()))) return false;
  c.q_weight = qw.data_ptr();
  c.k_weight = ptr(kw);
  c.param_dtype = code_of(qw.scalar_type());
  return true;
}
void run_rotary(const Tensor &q, const Tensor &k, gnnhwc_rotary_call &c, Tensor &qo, Tensor &ko) {
  const c10::DeviceGuard guard(q.device());
  const at::AutoDispatchBelowADInplaceOrView below;
  const OperatorRange range("gnop::rotary");
  qo = fresh(q.sizes(), q.scalar_type(), q);
  c.q = q.data_ptr();
  c.q_out = qo.data_ptr();
  put_strides(q, c.q_stride);
  put_strides(qo, c.q_out_stride);
  if (k.defined()) {
    ko = fresh(k.sizes(), k.scalar_type(), k);
    c.k = k.data_ptr();
    c.k_out = ko.data_ptr();
    put_strides(k, c.k_stride);
    put_strides(ko, c.k_out_stride);
  }
  check(abi.rotary(&c, stream_of(q)), "gnop::rotary");
}

struct RotaryNode : public torch::autograd::Function<RotaryNode> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext *ctx, const Tensor &q, const optional<Tensor> &k,
                                                const optional<Tensor> &qw, const optional<Tensor> &kw, const RotaryArgs *a, gnnhwc_rotary_call *c) {
    Tensor qo, ko;
    run_rotary(q, defined(k), *c, qo, ko);
    const bool norm = qw.has_value();
    ctx->save_for_backward({norm ? q : Tensor(), norm ? defined(k) : Tensor(), a->positions, a->frequencies, defined(qw), defined(kw)});
    ctx->saved_data["sections"] = a->sections;
    ctx->saved_data["interleaved"] = a->interleaved;
    ctx->saved_data["eps"] = a->eps;
    if (!k.has_value()) return {qo};
    return {qo, ko};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor q = saved[0], k = saved[1], qw = saved[4], kw = saved[5], gq = grads[0], gk = grads.size() > 1 ? grads[1] : Tensor();
    RotaryArgs a;
    a.positions = saved[2];
    a.frequencies = saved[3];
    a.sections = ctx->saved_data["sections"].toIntVector();
    a.interleaved = ctx->saved_data["interleaved"].toBool();
    a.eps = ctx->saved_data["eps"].toDouble();
    const bool has_k = gk.defined(), norm = qw.defined();
    const c10::Device device = gq.device();
    gnnhwc_rotary_call c = {};
    Tensor dq, dk, dqw, dkw;
    // (as for the norm: whatever is not plain goes through the operator)
    if (at::GradMode::is_enabled() || !ordinary_dispatch() || !heads_fit(gq, device) || (has_k && !like_q(gk, gq)) ||
        !rotary_call(gq, gk, a, c) || !put_weights(qw, kw, gq, has_k, c) ||
        (norm && (!like_q(q, gq) || q.size(2) != gq.size(2) || (has_k && (!k.defined() || !like_q(k, gk) || k.size(2) != gk.size(2)))))) {
      using Signature = std::tuple<Tensor, Tensor, Tensor, Tensor>(
          const Tensor &, const optional<Tensor> &, const optional<Tensor> &, const optional<Tensor> &, const Tensor &, const Tensor &, at::IntArrayRef,
          bool, const optional<Tensor> &, const optional<Tensor> &, double);
      const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("gnop::rotary_bwd", "").typed<Signature>();
      const auto opt = [](const Tensor &t) { return t.defined() ? optional<Tensor>(t) : std::nullopt; };
      std::tie(dq, dk, dqw, dkw) = op.call(gq, opt(gk), opt(q), opt(k), a.positions, a.frequencies, a.sections, a.interleaved, opt(qw), opt(kw), a.eps);
    } else {
      const c10::DeviceGuard guard(device);
      const at::AutoDispatchBelowADInplaceOrView below;
      const OperatorRange range("gnop::rotary_bwd");
      dq = fresh(gq.sizes(), gq.scalar_type(), gq);
      c.q_grad = gq.data_ptr();
      c.q_out = dq.data_ptr();
      put_strides(gq, c.q_grad_stride);
      put_strides(dq, c.q_out_stride);
      if (has_k) {
        dk = fresh(gk.sizes(), gk.scalar_type(), gk);
        c.k_grad = gk.data_ptr();
        c.k_out = dk.data_ptr();
        put_strides(gk, c.k_grad_stride);
        put_strides(dk, c.k_out_stride);
      }
      Tensor ws;
      size_t bytes = 0;
      if (norm) {
        c.q = q.data_ptr();
        put_strides(q, c.q_stride);
        dqw = fresh({c.head_dim}, qw.scalar_type(), qw);
        c.q_dweight = dqw.data_ptr();
        if (has_k) {
          c.k = k.data_ptr();
          put_strides(k, c.k_stride);
          dkw = fresh({c.head_dim}, kw.scalar_type(), kw);
          c.k_dweight = dkw.data_ptr();
        }
        bytes = abi.rotary_bwd_workspace_bytes(&c);
        ws = workspace(bytes, gq, "gnop::rotary_bwd");
      }
      check(abi.rotary_bwd(&c, ptr(ws), bytes, stream_of(gq)), "gnop::rotary_bwd");
    }
    return {dq, has_k ? dk : Tensor(), norm ? dqw : Tensor(), norm && has_k ? dkw : Tensor(), Tensor(), Tensor()};
  }
};

// rotary(q, k, positions, frequencies, sections, interleaved, q_weight, k_weight, eps) -> q', (q', k') or NotImplemented
PyObject *rotary(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  TORCH_CHECK(nargs == 9, "rotary takes 9 arguments");
  optional<Tensor> q_, k_, positions, frequencies, qw_, kw_;
  RotaryArgs a;
  if (!tensor_or_none(args[0], q_) || !q_.has_value() || !ordinary_thread() || !tensor_or_none(args[1], k_) || !tensor_or_none(args[2], positions) ||
      !positions.has_value() || !tensor_or_none(args[3], frequencies) || !frequencies.has_value() || !tensor_or_none(args[6], qw_) ||
      !tensor_or_none(args[7], kw_) || !PyBool_Check(args[5]) || !eps_of(args[8], a.eps))
    return decline();
  a.positions = *positions;
  a.frequencies = *frequencies;
  a.interleaved = args[5] == Py_True;
  if (args[4] == Py_None) {
    a.sections.push_back(a.frequencies.numel());
  } else {
    if (!PyTuple_CheckExact(args[4])) return decline();
    for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(args[4]); ++i) {
      PyObject *n = PyTuple_GET_ITEM(args[4], i);
      const int64_t v = PyLong_CheckExact(n) ? PyLong_AsLongLong(n) : -1;
      if (v < 0 || v > 65536) {
        PyErr_Clear();
        return decline();
      }
      a.sections.push_back(v);
    }
  }
  const Tensor q = *q_, k = defined(k_), qw = defined(qw_), kw = defined(kw_);
  gnnhwc_rotary_call c = {};
  if (code_of(q.scalar_type()) < 0 || !heads_fit(q, q.device()) || (k.defined() && !like_q(k, q)) || !rotary_call(q, k, a, c) ||
      !put_weights(qw, kw, q, k.defined(), c))
    return decline();
  const int64_t turning = 2 * c.section_end[c.axes - 1];
  if (c.head_dim % 2 || c.head_dim > 256 || (c.head_dim > 128 && (c.head_dim % 8 || turning % 8)) || turning > c.head_dim || turning < 1 ||
      q.numel() >= ((int64_t)1 << 33))
    return decline();  // sizes that the library may refuse: the general form says why
  Tensor qo, ko;
  {
    const WithoutGil released;
    if (wants_grad({q, k, qw, kw})) {
      const auto opt = [](const Tensor &t) { return t.defined() ? optional<Tensor>(t) : std::nullopt; };
      const auto out = RotaryNode::apply(q, opt(k), opt(qw), opt(kw), &a, &c);
      qo = out[0];
      if (out.size() > 1) ko = out[1];
    } else {
      run_rotary(q, k, c, qo, ko);
    }
  }
  if (!k.defined()) return THPVariable_Wrap(qo);
  return wrap_all({qo, ko});
  END_HANDLE_TH_ERRORS
}

// ---- gradient clipping ----
// clip_gradients(grads, max_norm, out or None, grad_scale, eps) -> total or NotImplemented; grads and out are lists
PyObject *clip_gradients(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  TORCH_CHECK(nargs == 5, "clip_gradients takes 5 arguments");
  if (!PyList_CheckExact(args[0]) || !PyFloat_CheckExact(args[1]) || !(args[2] == Py_None || PyList_CheckExact(args[2])) ||
      !PyFloat_CheckExact(args[3]) || !PyFloat_CheckExact(args[4]) || !ordinary_thread())
    return decline();
  const Py_ssize_t n = PyList_GET_SIZE(args[0]);
  const bool elsewhere = args[2] != Py_None;
  if (n == 0 || (elsewhere && PyList_GET_SIZE(args[2]) != n)) return decline();
  const double max_norm = PyFloat_AS_DOUBLE(args[1]), grad_scale = PyFloat_AS_DOUBLE(args[3]), eps = PyFloat_AS_DOUBLE(args[4]);
  std::vector<const void *> in((size_t)n);
  std::vector<void *> out(elsewhere ? (size_t)n : 0);
  std::vector<int64_t> sizes((size_t)n);
  std::vector<int> types((size_t)n), out_types(elsewhere ? (size_t)n : 0);
  std::vector<Tensor> written;  // their versions move on, as with any change in place
  written.reserve((size_t)n);
  Tensor first;
  bool all_double = true;
  const bool changes = elsewhere || grad_scale != 1.0 || max_norm < INFINITY;
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject *o = PyList_GET_ITEM(args[0], i);
    if (!THPVariable_CheckExact(o)) return decline();
    const Tensor &g = THPVariable_Unpack(o);
    if (i == 0) first = g;
    const int code = code_of(g.scalar_type());
    if (code < 0 || !plain(g, first.device()) || !g.is_non_overlapping_and_dense()) return decline();
    all_double = all_double && code == GNNHWC_F64;
    in[i] = g.data_ptr();
    sizes[i] = g.numel();
    types[i] = code;
    if (elsewhere) {
      PyObject *p = PyList_GET_ITEM(args[2], i);
      if (!THPVariable_CheckExact(p)) return decline();
      const Tensor &t = THPVariable_Unpack(p);
      const int out_code = code_of(t.scalar_type());
      // (elements are paired by their place in memory: the orders of dimensions have to agree)
      if (out_code < 0 || !plain(t, first.device()) || t.sizes() != g.sizes() || !t.is_non_overlapping_and_dense() ||
          !(t.strides() == g.strides() || (t.is_contiguous() && g.is_contiguous())))
        return decline();
      out[i] = t.data_ptr();
      out_types[i] = out_code;
      written.push_back(t);
    } else if (changes) {
      written.push_back(g);
    }
  }
  Tensor total;
  {
    const WithoutGil released;
    const c10::DeviceGuard guard(first.device());
    const at::AutoDispatchBelowADInplaceOrView below;
    const OperatorRange range("gnop::clip_gradients");
    total = fresh({}, all_double ? at::kDouble : at::kFloat, first);
    const size_t bytes = abi.clip_workspace_bytes(n);
    const Tensor ws = workspace(bytes, first, "clip_gradients");
    check(abi.clip(in.data(), elsewhere ? out.data() : nullptr, sizes.data(), types.data(), elsewhere ? out_types.data() : nullptr, n, max_norm, eps,
                   grad_scale, total.data_ptr(), code_of(total.scalar_type()), ws.data_ptr(), bytes, stream_of(first)),
          "clip_gradients");
    for (const Tensor &t : written)
      if (!t.is_inference()) torch::autograd::impl::bump_version(t);
  }
  return THPVariable_Wrap(total);
  END_HANDLE_TH_ERRORS
}

// ---- attention ----
// Whether the kernels read t where it is: (B, tokens, heads, D) with contiguous channels, rows whole 16 bytes apart.
bool rows16(const Tensor &t, const c10::Device &device, at::ScalarType type) {
  if (!plain(t, device) || t.dim() != 4 || t.scalar_type() != type || t.numel() == 0 || t.stride(3) != 1 || (uintptr_t)t.data_ptr() % 16) return false;
  const int64_t each = 16 / t.element_size();
  for (int i = 0; i < 3; ++i)
    if (t.size(i) != 1 && t.stride(i) % each) return false;
  return t.size(1) == 1 || t.stride(1) * t.element_size() < (int64_t)1 << 25;
}
bool window_call(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &lengths, gnnhwc_window_call &c) {
  const c10::Device device = q.device();
  const at::ScalarType type = q.scalar_type();
  const int code = code_of(type);
  if (code < 0 || code == GNNHWC_F64 || !rows16(q, device, type) || !rows16(k, device, type) || !rows16(v, device, type)) return false;
  if (k.size(0) != q.size(0) || k.size(3) != q.size(3) || v.sizes() != k.sizes() || q.size(2) % k.size(2) || q.size(3) % 8 ||
      q.size(3) > (code == GNNHWC_F32 ? 128 : 256))
    return false;
  if (lengths.defined()) {
    if (!plain(lengths, device) || lengths.dim() != 1 || lengths.size(0) != q.size(0) || !lengths.is_contiguous()) return false;
    if (lengths.scalar_type() != at::kInt && lengths.scalar_type() != at::kLong) return false;
    c.lengths = lengths.data_ptr();
    c.length_type = lengths.scalar_type() == at::kLong;
  }
  c.q = q.data_ptr();
  c.k = k.data_ptr();
  c.v = v.data_ptr();
  put_strides(q, c.q_stride);
  put_strides(k, c.k_stride);
  put_strides(v, c.v_stride);
  c.batch = q.size(0);
  c.tokens = q.size(1);
  c.keys = k.size(1);
  c.heads = q.size(2);
  c.kv_heads = k.size(2);
  c.head_dim = q.size(3);
  c.dtype = code;
  return true;
}
// What the backward reads beside the forward's tensors, in one allocation: lse, then, in 16 bits, what rounding left of out.
struct WindowKept {
  int64_t lse_bytes, bytes;
  explicit WindowKept(const Tensor &q) {
    lse_bytes = (q.size(0) * q.size(1) * q.size(2) * 4 + 15) / 16 * 16;
    bytes = lse_bytes + (q.scalar_type() == at::kFloat ? 0 : q.numel() * 2);
  }
  void put(const Tensor &kept, gnnhwc_window_call &c) const {
    c.lse = (float *)kept.data_ptr();
    c.out_rest = bytes > lse_bytes ? (char *)kept.data_ptr() + lse_bytes : nullptr;
  }
};
void run_window(const Tensor &q, gnnhwc_window_call &c, Tensor &out, Tensor *kept) {
  const c10::DeviceGuard guard(q.device());
  const at::AutoDispatchBelowADInplaceOrView below;
  const OperatorRange range("gnop::window_attention");
  out = fresh(q.sizes(), q.scalar_type(), q);
  c.out = out.data_ptr();
  put_strides(out, c.out_stride);
  if (kept) {
    const WindowKept parts(q);
    *kept = fresh({parts.bytes}, at::kByte, q);
    parts.put(*kept, c);
  }
  const size_t bytes = abi.window_workspace_bytes(&c);
  Tensor ws;
  if (bytes != GNNHWC_WINDOW_NO_WORKSPACE) ws = workspace(bytes, q, "gnop::window_attention");
  check(abi.window(&c, ptr(ws), bytes, stream_of(q)), "gnop::window_attention");
}

struct WindowNode : public torch::autograd::Function<WindowNode> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &v,
                                                const optional<Tensor> &lengths, gnnhwc_window_call *c) {
    Tensor out, kept;
    run_window(q, *c, out, &kept);
    ctx->save_for_backward({q, k, v, out, kept, defined(lengths)});
    ctx->saved_data["call"] = std::vector<int64_t>{c->window, c->sinks, c->causal};
    ctx->saved_data["scale"] = c->scale;
    return {out};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor q = saved[0], k = saved[1], v = saved[2], out = saved[3], kept = saved[4], lengths = saved[5], dout = grads[0];
    const c10::Device device = dout.device();
    gnnhwc_window_call c = {};
    const auto numbers = ctx->saved_data["call"].toIntVector();
    c.window = numbers[0];
    c.sinks = numbers[1];
    c.causal = numbers[2];
    c.scale = ctx->saved_data["scale"].toDouble();
    const WindowKept parts(q);
    Tensor dq, dk, dv;
    // (as for the norm: whatever is not plain goes through the operator)
    if (at::GradMode::is_enabled() || !ordinary_dispatch() || !plain(q, device) || !window_call(q, k, v, lengths, c) ||
        !rows16(dout, device, q.scalar_type()) || dout.sizes() != q.sizes() || !rows16(out, device, q.scalar_type()) || out.sizes() != q.sizes() ||
        !plain(kept, device) || !kept.is_contiguous() || kept.scalar_type() != at::kByte || kept.numel() != parts.bytes || (uintptr_t)kept.data_ptr() % 16) {
      TORCH_CHECK(kept.dim() == 1 && kept.numel() == parts.bytes && kept.scalar_type() == at::kByte, "window_attention: a saved tensor came back as another");
      const Tensor lse = kept.narrow(0, 0, q.size(0) * q.size(1) * q.size(2) * 4).view(at::kFloat).view({q.size(0), q.size(2), q.size(1)});
      const Tensor rest = parts.bytes > parts.lse_bytes ? kept.narrow(0, parts.lse_bytes, q.numel() * 2).view(q.scalar_type()).view(q.sizes())
                                                        : at::empty({0}, q.options());
      using Signature = std::tuple<Tensor, Tensor, Tensor>(const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &,
                                                           const Tensor &, const optional<Tensor> &, int64_t, int64_t, bool, double);
      const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("gnop::window_attention_bwd", "").typed<Signature>();
      std::tie(dq, dk, dv) = op.call(dout, q, k, v, out, lse, rest, lengths.defined() ? optional<Tensor>(lengths) : std::nullopt, c.window, c.sinks, c.causal, c.scale);
    } else {
      const c10::DeviceGuard guard(device);
      const at::AutoDispatchBelowADInplaceOrView below;
      const OperatorRange range("gnop::window_attention_bwd");
      dq = fresh(q.sizes(), q.scalar_type(), q);
      dk = fresh(k.sizes(), k.scalar_type(), k);
      dv = fresh(v.sizes(), v.scalar_type(), v);
      c.out = out.data_ptr();
      parts.put(kept, c);
      c.out_grad = dout.data_ptr();
      c.q_grad = dq.data_ptr();
      c.k_grad = dk.data_ptr();
      c.v_grad = dv.data_ptr();
      put_strides(out, c.out_stride);
      put_strides(dout, c.out_grad_stride);
      put_strides(dq, c.q_grad_stride);
      put_strides(dk, c.k_grad_stride);
      put_strides(dv, c.v_grad_stride);
      const size_t bytes = abi.window_bwd_workspace_bytes(&c);
      const Tensor ws = workspace(bytes, q, "gnop::window_attention_bwd");
      check(abi.window_bwd(&c, ws.data_ptr(), bytes, stream_of(q)), "gnop::window_attention_bwd");
    }
    return {dq, dk, dv, Tensor(), Tensor()};
  }
};

// A Python integer that is exactly one and not negative, or false.
bool whole_number(PyObject *o, int64_t &v) {
  if (!PyLong_CheckExact(o)) return false;
  v = PyLong_AsLongLong(o);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return v >= 0;
}

// window_attention(q, k, v, lengths, window or None, sinks, causal, at_end, scale or None) -> out or NotImplemented
PyObject *window_attention(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  TORCH_CHECK(nargs == 9, "window_attention takes 9 arguments");
  optional<Tensor> q_, k_, v_, lengths_;
  if (!tensor_or_none(args[0], q_) || !q_.has_value() || !ordinary_thread() || !tensor_or_none(args[1], k_) || !k_.has_value() ||
      !tensor_or_none(args[2], v_) || !v_.has_value() || !tensor_or_none(args[3], lengths_) || !PyBool_Check(args[6]) || !PyBool_Check(args[7]))
    return decline();
  const Tensor q = *q_, k = *k_, v = *v_, lengths = defined(lengths_);
  gnnhwc_window_call c = {};
  c.window = -1;
  if (args[4] != Py_None && !whole_number(args[4], c.window)) return decline();
  if (!whole_number(args[5], c.sinks) || !window_call(q, k, v, lengths, c)) return decline();
  c.causal = args[6] == Py_True;
  c.at_end = args[7] == Py_True;
  c.scale = 1.0 / std::sqrt((double)c.head_dim);
  if (args[8] != Py_None) {
    if (!PyFloat_CheckExact(args[8])) return decline();
    c.scale = PyFloat_AS_DOUBLE(args[8]);
  }
  const bool differentiates = wants_grad({q, k, v});
  // (sizes that the library may refuse: the general form says why)
  if (!(c.scale > 1e-30 && c.scale < 1e30) || (!c.at_end && c.tokens > c.keys) || (c.at_end && differentiates) || c.keys > (1 << 30) || c.tokens > (1 << 30) ||
      c.heads > 65535 || c.batch * c.heads * (c.tokens / 128 + 1) > 1 << 22)
    return decline();
  Tensor out;
  {
    const WithoutGil released;
    if (differentiates) out = WindowNode::apply(q, k, v, lengths_, &c)[0];
    else run_window(q, c, out, nullptr);
  }
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// ---- dropout ----
struct DropoutCall {
  double p = 0;
  uint64_t seed = 0, offset = 0;
  Tensor seed_at;  // possibly undefined
};
Tensor run_dropout(const Tensor &x, const Tensor &residual, const DropoutCall &c) {
  const c10::DeviceGuard guard(x.device());
  const at::AutoDispatchBelowADInplaceOrView below;
  const OperatorRange range("gnop::dropout");
  Tensor y = fresh(x.sizes(), x.scalar_type(), x);
  check(abi.dropout(x.data_ptr(), ptr(residual), y.data_ptr(), x.numel(), c.p, c.seed, (const int64_t *)ptr(c.seed_at), c.offset,
                    code_of(x.scalar_type()), stream_of(x)),
        "gnop::dropout");
  return y;
}
struct DropoutNode : public torch::autograd::Function<DropoutNode> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext *ctx, const Tensor &x, const optional<Tensor> &residual,
                                                const DropoutCall *c) {
    ctx->save_for_backward({c->seed_at});
    ctx->saved_data["p"] = c->p;
    ctx->saved_data["seed"] = (int64_t)c->seed;
    ctx->saved_data["offset"] = (int64_t)c->offset;
    ctx->saved_data["residual"] = residual.has_value();
    return {run_dropout(x, defined(residual), *c)};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads) {
    const Tensor dy = grads[0];
    const bool residual = ctx->saved_data["residual"].toBool();
    DropoutCall c;
    c.p = ctx->saved_data["p"].toDouble();
    c.seed = (uint64_t)ctx->saved_data["seed"].toInt();
    c.offset = (uint64_t)ctx->saved_data["offset"].toInt();
    c.seed_at = ctx->get_saved_variables()[0];
    Tensor dx;
    if (ctx->needs_input_grad(0)) {
      if (at::GradMode::is_enabled() || !ordinary_dispatch() || !plain(dy, dy.device()) || !dy.is_contiguous() || dy.numel() == 0 ||
          code_of(dy.scalar_type()) < 0) {
        using Signature = Tensor(const Tensor &, const optional<Tensor> &, double, int64_t, const optional<Tensor> &, int64_t);
        const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("gnop::dropout", "").typed<Signature>();
        dx = op.call(dy, std::nullopt, c.p, (int64_t)c.seed, c.seed_at.defined() ? optional<Tensor>(c.seed_at) : std::nullopt, (int64_t)c.offset);
      } else {
        dx = run_dropout(dy, Tensor(), c);
      }
    }
    return {dx, residual ? dy : Tensor(), Tensor()};
  }
};

// dropout(x, residual, p, seed (integer of 64 bits or tensor), offset) -> y or NotImplemented
PyObject *dropout(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  TORCH_CHECK(nargs == 5, "dropout takes 5 arguments");
  optional<Tensor> x_, residual_;
  DropoutCall c;
  if (!tensor_or_none(args[0], x_) || !x_.has_value() || !ordinary_thread() || !tensor_or_none(args[1], residual_) || !PyFloat_CheckExact(args[2]))
    return decline();
  const Tensor x = *x_, residual = defined(residual_);
  const auto fits = [&](const Tensor &t) {
    return plain(t, x.device()) && t.is_contiguous() && t.scalar_type() == x.scalar_type() && t.sizes() == x.sizes();
  };
  if (code_of(x.scalar_type()) < 0 || !fits(x) || x.numel() == 0 || x.numel() > (int64_t)1 << 34 || (residual.defined() && !fits(residual))) return decline();
  c.p = PyFloat_AS_DOUBLE(args[2]);
  int64_t seed = 0, offset = 0;
  if (!(c.p >= 0 && c.p <= 1) || !whole_number(args[4], offset)) return decline();
  if (!whole_number(args[3], seed)) {
    optional<Tensor> seed_at;
    if (args[3] == Py_None || !tensor_or_none(args[3], seed_at)) return decline();
    if (!plain(*seed_at, x.device()) || seed_at->scalar_type() != at::kLong || seed_at->numel() != 1) return decline();
    c.seed_at = *seed_at;
    seed = 0;
  }
  c.seed = (uint64_t)seed;
  c.offset = (uint64_t)offset;
  Tensor y;
  {
    const WithoutGil released;
    if (wants_grad({x, residual})) y = DropoutNode::apply(x, residual_, &c)[0];
    else y = run_dropout(x, residual, c);
  }
  return THPVariable_Wrap(y);
  END_HANDLE_TH_ERRORS
}

// bind_tokens(address, ...): the C ABI's functions in the order of Entry.
PyObject *bind_tokens(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  void **slot = reinterpret_cast<void **>(&abi);
  constexpr Py_ssize_t kSlots = sizeof(Entry) / sizeof(void *);
  if (nargs != kSlots) {
    PyErr_SetString(PyExc_TypeError, "bind_tokens: one address per entry point");
    return nullptr;
  }
  for (Py_ssize_t i = 0; i < kSlots; ++i) {
    slot[i] = PyLong_AsVoidPtr(args[i]);
    if (!slot[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "bind_tokens: null address");
      return nullptr;
    }
  }
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"rms_norm", (PyCFunction)(void (*)(void))rms_norm, METH_FASTCALL,
     "rms_norm(x, weight, eps, residual, return_sum) -> y, (y, s) or NotImplemented"},
    {"rms_norm_quant", (PyCFunction)(void (*)(void))rms_norm_quant, METH_FASTCALL,
     "rms_norm_quant(x, weight, eps, residual, return_sum, out_dtype, block) -> (q, scales), (q, scales, s) or NotImplemented"},
    {"rotary", (PyCFunction)(void (*)(void))rotary, METH_FASTCALL,
     "rotary(q, k, positions, frequencies, sections, interleaved, q_weight, k_weight, eps) -> q', (q', k') or NotImplemented"},
    {"clip_gradients", (PyCFunction)(void (*)(void))clip_gradients, METH_FASTCALL,
     "clip_gradients(grads, max_norm, out, grad_scale, eps) -> total or NotImplemented"},
    {"window_attention", (PyCFunction)(void (*)(void))window_attention, METH_FASTCALL,
     "window_attention(q, k, v, lengths, window, sinks, causal, at_end, scale) -> out or NotImplemented"},
    {"dropout", (PyCFunction)(void (*)(void))dropout, METH_FASTCALL, "dropout(x, residual, p, seed, offset) -> y or NotImplemented"},
    {"bind_tokens", (PyCFunction)(void (*)(void))bind_tokens, METH_FASTCALL, "bind_tokens(*addresses): the C ABI's entry points"},
    {nullptr, nullptr, 0, nullptr}};

}  // namespace

int gn_torch::add_token_methods(PyObject *module) { return PyModule_AddFunctions(module, methods); }
