// What the extension module's functions share.
#pragma once
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/ajq_serve.h"

namespace native {

// a tensor (or parameter) of the plain kind on the current device, or null
inline const at::Tensor* plain(PyObject* object) {
  if (!THPVariable_CheckExact(object)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(object);
  const c10::DispatchKeySet special({c10::DispatchKey::Python, c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper,
                                     c10::DispatchKey::Functionalize, c10::DispatchKey::Conjugate, c10::DispatchKey::Negative,
                                     c10::DispatchKey::ZeroTensor, c10::DispatchKey::Named});
  return t.is_cuda() && t.layout() == at::kStrided && !t.key_set().has_any(special) ? &t : nullptr;
}

// other threads run while the allocator and the runtime do (a full queue makes a launch wait)
struct WithoutInterpreter {
  PyThreadState* state = PyEval_SaveThread();
  ~WithoutInterpreter() { PyEval_RestoreThread(state); }
};

// whether a mode wants to see the operators
inline bool watched() { return c10::impl::TorchDispatchModeTLS::any_modes_set() || at::impl::torch_function_mode_enabled(); }

// Reads a call's arguments one after the other; `ok` falls at the first that is not as expected.
struct Arguments {
  PyObject* const* args;
  c10::DeviceIndex device = -1;
  bool ok = true;
  at::Tensor held[16];   // references, while the interpreter runs other threads
  int holds = 0;

  const at::Tensor* tensor(int i) {
    if (!ok) return nullptr;
    const at::Tensor* t = plain(args[i]);
    if (t == nullptr || (device >= 0 && t->device().index() != device)) {
      ok = false;
      return nullptr;
    }
    device = t->device().index();
    held[holds] = *t;
    return &held[holds++];
  }
  const at::Tensor* optional(int i) { return args[i] == Py_None ? nullptr : tensor(i); }
  int64_t number(int i) {
    if (!ok || !PyLong_CheckExact(args[i])) {
      ok = false;
      return 0;
    }
    const int64_t n = PyLong_AsLongLong(args[i]);
    if (n == -1 && PyErr_Occurred()) {
      PyErr_Clear();
      ok = false;
    }
    return n;
  }
  void need(bool condition) { ok = ok && condition; }

  static bool known(at::ScalarType type) { return type == at::kFloat || type == at::kBFloat16; }
  static int flag(at::ScalarType type) { return type == at::kBFloat16 ? AJQS_BF16 : AJQS_F32; }
  // int64, contiguous, `count` of them
  const int64_t* whole(const at::Tensor* t, int64_t count) {
    if (!ok || t == nullptr) return nullptr;
    need(t->scalar_type() == at::kLong && t->numel() == count && t->is_contiguous());
    return ok ? t->const_data_ptr<int64_t>() : nullptr;
  }
  const float* floats(const at::Tensor* t, at::IntArrayRef shape) {
    if (!ok || t == nullptr) return nullptr;
    need(t->scalar_type() == at::kFloat && t->sizes() == shape && t->is_contiguous());
    return ok ? t->const_data_ptr<float>() : nullptr;
  }
  void caches(const at::Tensor* keys, const at::Tensor* values) {
    if (!ok) return;
    need(keys->dim() == 4 && keys->sizes() == values->sizes() && keys->strides() == values->strides() && known(keys->scalar_type()) &&
         values->scalar_type() == keys->scalar_type());
    need(ok && keys->stride(3) == 1 && keys->stride(2) == keys->size(3));
    for (int d = 0; ok && d < 4; ++d) need(keys->size(d) >= 1 && keys->size(d) <= INT32_MAX);
  }
};

inline int as_int(int64_t n) { return (int)n; }
inline bool fits(int64_t n) { return n >= 0 && n <= INT32_MAX; }

// native_serve.cpp
PyObject* norm_rope(PyObject*, PyObject* const* args, Py_ssize_t count);
PyObject* shared_prefix_attention(PyObject*, PyObject* const* args, Py_ssize_t count);
PyObject* adjust_logits(PyObject*, PyObject* const* args, Py_ssize_t count);
PyObject* bind_serve(PyObject*, PyObject* const* args, Py_ssize_t count);
// native_draft.cpp
PyObject* tree_attention(PyObject*, PyObject* const* args, Py_ssize_t count);
PyObject* keep_rows(PyObject*, PyObject* const* args, Py_ssize_t count);
PyObject* token_log_probs(PyObject*, PyObject* const* args, Py_ssize_t count);
PyObject* follow_drafts(PyObject*, PyObject* const* args, Py_ssize_t count);
PyObject* bind_draft(PyObject*, PyObject* const* args, Py_ssize_t count);

}  // namespace native
