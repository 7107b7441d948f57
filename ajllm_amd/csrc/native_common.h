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

// native_serve.cpp
PyObject* norm_rope(PyObject*, PyObject* const* args, Py_ssize_t count);
PyObject* shared_prefix_attention(PyObject*, PyObject* const* args, Py_ssize_t count);
PyObject* adjust_logits(PyObject*, PyObject* const* args, Py_ssize_t count);
PyObject* bind_serve(PyObject*, PyObject* const* args, Py_ssize_t count);

}  // namespace native
