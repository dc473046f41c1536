// What the eager calls of gn_torch.cpp and gn_tokens_torch.cpp share: which tensors and threads are ordinary, dtype codes,
// the stream, and the scopes of a call.
#pragma once
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/record_function.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/gnnhwc.h"

namespace gn_torch {

using at::Tensor;
using std::optional;

inline int code_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return GNNHWC_F32;
    case at::kDouble: return GNNHWC_F64;
    case at::kHalf: return GNNHWC_F16;
    case at::kBFloat16: return GNNHWC_BF16;
    default: return -1;
  }
}
inline bool is_half(at::ScalarType t) { return t == at::kHalf || t == at::kBFloat16; }

inline void *stream_of(const Tensor &x) { return (void *)c10::hip::getCurrentHIPStream(x.device().index()).stream(); }

// The operator's name in torch's profiler, around one call.
class OperatorRange {
 public:
  explicit OperatorRange(const char *what) : range_(at::RecordScope::FUNCTION) {
    if (range_.isActive()) range_.before(what);
  }

 private:
  at::RecordFunction range_;
};

// Dispatch keys of a plain device tensor; any other key (a subclass, a transform's wrapper, a lazy conjugate ...) declines.
inline const c10::DispatchKeySet &plain_keys() {
  static const c10::DispatchKeySet keys = c10::DispatchKeySet(c10::DispatchKey::CUDA) |
                                          c10::DispatchKeySet(c10::DispatchKey::AutogradCUDA) |
                                          c10::DispatchKeySet(c10::DispatchKey::ADInplaceOrView) |
                                          c10::DispatchKeySet(c10::DispatchKey::AutocastCUDA);
  return keys;
}
// Keys that are switched on for every thread, or by autocast (which has no rule for this operation).
inline const c10::DispatchKeySet &plain_tls() {
  static const c10::DispatchKeySet keys =
      c10::default_included_set | c10::autocast_dispatch_keyset | c10::DispatchKeySet(c10::DispatchKey::ADInplaceOrView);
  return keys;
}
// (by the bits: the sets' difference keeps the bits of the backends)
inline bool only(c10::DispatchKeySet keys, c10::DispatchKeySet allowed) { return (keys.raw_repr() & ~allowed.raw_repr()) == 0; }
inline bool ordinary_dispatch() {
  return !c10::impl::TorchDispatchModeTLS::any_modes_set() && only(c10::impl::tls_local_dispatch_key_set().included_, plain_tls());
}
inline bool ordinary_thread() { return at::impl::PythonTorchFunctionTLS::stack_len() == 0 && ordinary_dispatch(); }
inline bool plain(const Tensor &t, const c10::Device &device) {
  return t.defined() && t.is_cuda() && t.device() == device && t.layout() == at::kStrided && only(t.key_set(), plain_keys()) &&
         !t._fw_grad(0).defined();
}

// While it lives, other Python threads run: allocations may have to wait for the device, launches for a full queue or for
// another thread's.  (Saved-tensor hooks and operators implemented in Python take the lock again by themselves.)
class WithoutGil {
 public:
  WithoutGil() : state_(PyEval_SaveThread()) {}
  ~WithoutGil() { PyEval_RestoreThread(state_); }
  WithoutGil(const WithoutGil &) = delete;
  WithoutGil &operator=(const WithoutGil &) = delete;

 private:
  PyThreadState *state_;
};
inline bool needs_grad(const optional<Tensor> &t) { return t.has_value() && t->requires_grad(); }

// None -> no value; an exact torch.Tensor / Parameter -> its tensor; anything else -> false.
inline bool tensor_or_none(PyObject *o, optional<Tensor> &t) {
  if (o == Py_None) return true;
  if (!THPVariable_CheckExact(o)) return false;
  t = THPVariable_Unpack(o);
  return true;
}

// The functions of gn_tokens_torch.cpp, added to the module; -1 with a Python error set on failure.
int add_token_methods(PyObject *module);

}  // namespace gn_torch
