// Shared by the operators' host sides (host_native.cpp, host_wide.cpp): torch tensors as addresses, strides and codes of the C interface, and
// the arguments of Python calls.
#pragma once

#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/autocast_mode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/InferenceMode.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <array>
#include <cstring>
#include <memory>
#include <mutex>
#include <optional>
#include <vector>

#include "nf_cdna4.h"

namespace {  // each file its own copy: nothing of this is exported

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// ------------------------------------------------------------------------------------------------ pieces
int code_of(at::ScalarType t) {
  return t == at::kFloat ? NF_F32 : t == at::kHalf ? NF_F16 : t == at::kBFloat16 ? NF_BF16 : -1;
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// (a negated view, the imaginary part of a conjugate, holds its values with the other sign: its memory is not read as it is)
Tensor resolved(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }

Tensor contiguous(const Tensor& t) { return t.defined() ? resolved(t).contiguous() : t; }

void check(int rc, const char* what) { TORCH_CHECK(rc == 0, what, " failed (code ", rc, "): ", nf_last_error()); }

Tensor scratch(int64_t bytes, const Tensor& like) {
  return bytes > 0 ? at::empty({bytes}, like.options().dtype(at::kByte)) : Tensor();
}

// A tensor as rows of `width`: address, row stride and count.  Rows that overlap (an expanded tensor has row stride 0) or a
// strided inner dimension are copied.
struct Rows {
  Tensor hold;
  void* p;
  int64_t n, stride;
  Rows(const Tensor& t, int64_t width) : hold(resolved(t)), n(t.numel() / width), stride(width) {
    if (!hold.is_contiguous()) {
      hold = hold.reshape({-1, width});
      if (hold.stride(1) != 1 || (n > 1 && hold.stride(0) < width)) hold = hold.contiguous();
      stride = hold.stride(0);
    }
    p = hold.data_ptr();
  }
};

// The gradients that a kernel computed have no graph.  Where one is asked for (create_graph), each of them that depends on something which requires a gradient gets a
// node that raises: a second derivative is refused instead of lost.  The node leads to what the gradient depends on, so that a backward for
// these tensors alone comes to it, too.
struct Once {
  const char* name;
  std::shared_ptr<torch::autograd::Node> node;  // whose backward runs (none: no graph is asked for); its edges are the forward's tensors in their order
  explicit Once(const char* what) : name(what), node(at::GradMode::is_enabled() ? torch::autograd::get_current_node() : nullptr) {}
  // `inputs`: the numbers of the forward's tensors that g depends on; `grads`: the upstream gradients
  void mark(const Tensor& g, std::initializer_list<int> inputs, std::initializer_list<Tensor> grads) const {
    if (node == nullptr || !g.defined()) return;
    torch::autograd::edge_list edges;
    for (const int i : inputs)
      if ((uint32_t)i < node->num_outputs() && node->next_edge(i).is_valid()) edges.push_back(node->next_edge(i));
    for (const Tensor& t : grads)
      if (t.defined() && t.requires_grad()) edges.push_back(torch::autograd::impl::gradient_edge(t));
    if (edges.empty()) return;
    const std::shared_ptr<torch::autograd::Node> raises(
        new torch::autograd::Error(std::string(name) + " is differentiable once: its gradients have no derivatives", std::move(edges)), torch::autograd::deleteNode);
    torch::autograd::set_history(g, raises);
  }
};

// ------------------------------------------------------------------------------------------------ Python
// A plain GPU tensor: no subclass, no wrapper of a function transform, no tangent of a forward-mode derivative (the kernels have no
// such derivative: the autograd Function refuses it), a floating type the kernels know.
bool plain(PyObject* o, Tensor* t) {
  if (!THPVariable_CheckTypeExact(Py_TYPE(o))) return false;
  *t = THPVariable_Unpack(o);
  const auto keys = t->key_set();
  return t->is_cuda() && t->layout() == at::kStrided && !keys.has(c10::DispatchKey::FuncTorchBatched) &&
         !keys.has(c10::DispatchKey::FuncTorchGradWrapper) && !keys.has(c10::DispatchKey::Functionalize) && !keys.has(c10::DispatchKey::Python) &&
         !t->is_conj() && !t->is_neg() && !t->_fw_grad(/*level=*/0).defined();
}

bool plain_or_none(PyObject* o, std::optional<Tensor>* t) {
  if (o == Py_None) return true;
  Tensor v;
  if (!plain(o, &v)) return false;
  *t = std::move(v);
  return true;
}

// A dispatch or function mode, a function transform (vmap, grad, jvp: the autograd Functions refuse them), or the tracer, which records
// an autograd Function but would see nothing of a launch made here.
bool modes_active() {
  return c10::impl::TorchDispatchModeTLS::any_modes_set() || at::impl::torch_function_mode_enabled() || torch::jit::tracer::isTracing() ||
         c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode);
}

bool autocast() { return at::autocast::is_autocast_enabled(at::kCUDA); }

bool as_int(PyObject* o, int64_t* v) {
  if (!PyLong_CheckExact(o)) return false;
  int overflow = 0;
  *v = PyLong_AsLongLongAndOverflow(o, &overflow);
  return overflow == 0;
}

bool as_double(PyObject* o, double* v) {
  if (!PyFloat_CheckExact(o) && !PyLong_CheckExact(o)) return false;
  *v = PyFloat_AsDouble(o);
  if (*v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}

int activation(PyObject* o, bool gelu) {
  if (!PyUnicode_Check(o)) return -1;
  const char* s = PyUnicode_AsUTF8(o);
  if (s == nullptr) {
    PyErr_Clear();
    return -1;
  }
  if (!strcmp(s, "relu")) return NF_ACT_RELU;
  if (!strcmp(s, "silu")) return NF_ACT_SILU;
  if (!strcmp(s, "relu2")) return NF_ACT_RELU2;
  if (!strcmp(s, "none")) return NF_ACT_NONE;
  return gelu && !strcmp(s, "gelu") ? NF_ACT_GELU : -1;
}

PyObject* wrap(const Tensor& t) { return THPVariable_Wrap(t); }

PyObject* wrap_list(const variable_list& v) {
  PyObject* r = PyTuple_New((Py_ssize_t)v.size());
  if (r == nullptr) return nullptr;
  for (size_t i = 0; i < v.size(); ++i) {
    PyObject* o = v[i].defined() ? wrap(v[i]) : Py_NewRef(Py_None);
    if (o == nullptr) {
      Py_DECREF(r);
      return nullptr;
    }
    PyTuple_SET_ITEM(r, (Py_ssize_t)i, o);
  }
  return r;
}

Tensor tensor_arg(PyObject* o) { return o == Py_None ? Tensor() : THPVariable_Unpack(o); }

#define ENTRY(f) {#f, (PyCFunction)(void (*)(void))f, METH_FASTCALL, nullptr}
#define NARGS(k) TORCH_CHECK(n == (k), "expected ", (k), " arguments, got ", n)


}  // namespace
