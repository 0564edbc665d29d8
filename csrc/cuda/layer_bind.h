// Argument handling shared by the bindings of the dense and norm kernels.
#pragma once
#include <torch/extension.h>

#include <ATen/autocast_mode.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <string>

#include "dense.h"

namespace ngl {
namespace bind {

using OptTensor = c10::optional<torch::Tensor>;

inline void ck(cudaError_t e, const char* what) { TORCH_CHECK(e == cudaSuccess, what, ": ", cudaGetErrorString(e)); }

inline int sm_count(int device) {
  static int cached[64] = {0};
  if (device >= 0 && device < 64 && cached[device]) return cached[device];
  int v = 0;
  ck(cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, device), "multiprocessor count");
  if (device >= 0 && device < 64) cached[device] = v;
  return v;
}

inline int type_of(torch::ScalarType t) {
  if (t == torch::kFloat32) return dense::kF32;
  if (t == torch::kBFloat16) return dense::kBF16;
  if (t == torch::kHalf) return dense::kF16;
  if (t == at::kFloat8_e4m3fn) return dense::kE4M3;
  return -1;
}
inline bool is_half(torch::ScalarType t) { return t == torch::kBFloat16 || t == torch::kHalf; }

// Numbers and sizes for messages, as strings: an extension whose C++ library is
// linked statically cannot stream numbers through torch's message builder.
inline std::string text(int64_t v) { return std::to_string(v); }
inline std::string text(at::IntArrayRef v) {
  std::string s = "[";
  for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + std::to_string(v[i]);
  return s + "]";
}

inline void need_cuda(const torch::Tensor& t, const torch::Tensor& like, const char* what) {
  TORCH_CHECK(t.is_cuda(), what, " must be a CUDA tensor (there is no CPU path)");
  TORCH_CHECK(t.device() == like.device(), what, " is on cuda:", text(t.get_device()), ", x on cuda:",
              text(like.get_device()));
}

// [rows, cols] view of a tensor whose rows lie `ld` elements apart with
// contiguous columns; a copy where the strides allow no such view.
struct Rows {
  torch::Tensor t;  // keeps the memory alive
  int64_t ld;
  const void* p() const { return t.data_ptr(); }
};
inline Rows rows_of(const torch::Tensor& x, int64_t rows, int64_t cols) {
  torch::Tensor t = x.dim() == 2 ? x : x.reshape({rows, cols});
  if ((cols > 1 && t.stride(1) != 1) || (rows > 1 && t.stride(0) < cols)) t = t.contiguous();
  return {t, rows > 1 ? t.stride(0) : cols};
}

inline bool wants_grad(const torch::Tensor& t) { return t.requires_grad(); }
inline bool wants_grad(const OptTensor& t) { return t.has_value() && t->requires_grad(); }

inline bool has_tangent(const torch::Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }
inline bool has_tangent(const OptTensor& t) { return t.has_value() && has_tangent(*t); }
// The calls here do not go through the dispatcher, so what watches it does not
// see them: a tangent would be lost without a word, and a trace would hold the
// output as a constant.
template <typename... T>
void seen_by_all(const char* what, const T&... t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!(has_tangent(t) || ...), what, " has no forward-mode derivative");
  TORCH_CHECK_NOT_IMPLEMENTED(!torch::jit::tracer::isTracing(), what, " cannot be traced by torch.jit.trace");
}

// New tensors without the dispatcher's cost (a call of few rows is bound by
// the host).
inline torch::Tensor new_cuda(at::IntArrayRef sizes, at::ScalarType t, const torch::Tensor& like) {
  return at::detail::empty_cuda(sizes, t, like.device(), c10::nullopt);
}

// Gradients have no gradients of their own: one asked for raises.
inline torch::autograd::variable_list once(torch::autograd::variable_list grads, const char* what) {
  if (!at::GradMode::is_enabled()) return grads;
  torch::autograd::variable_list in;
  for (auto& g : grads)
    if (g.defined()) in.push_back(g.detach().set_requires_grad(true));
  auto fn = std::make_shared<torch::autograd::DelayedError>(
      std::string("no second derivative of ") + what, (int64_t)in.size());
  auto out = (*fn)(std::move(in));
  size_t i = 0;
  for (auto& g : grads)
    if (g.defined()) g = out[i++];
  return grads;
}

// ---- arguments of the functions that Python calls without pybind: its
// conversion of eight arguments takes 3 us, half of a call of one token.
inline const torch::Tensor& tensor_arg(PyObject* o, const char* what) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), what, " must be a torch.Tensor, not ", Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}
inline OptTensor opt_tensor_arg(PyObject* o, const char* what) {
  if (o == Py_None) return c10::nullopt;
  return tensor_arg(o, what);
}
inline c10::optional<at::ScalarType> opt_dtype_arg(PyObject* o, const char* what) {
  if (o == Py_None) return c10::nullopt;
  TORCH_CHECK_TYPE(THPDtype_Check(o), what, " must be a torch.dtype, not ", Py_TYPE(o)->tp_name);
  return reinterpret_cast<THPDtype*>(o)->scalar_type;
}
inline double float_arg(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}
inline int64_t int_arg(PyObject* o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}
inline void count_args(Py_ssize_t n, Py_ssize_t want, const char* what) {
  TORCH_CHECK_TYPE(n == want, what, " takes ", text(want), " arguments");
}
inline PyObject* wrap_all(const std::vector<torch::Tensor>& v) {
  PyObject* t = PyTuple_New((Py_ssize_t)v.size());
  if (t == nullptr) throw python_error();
  for (size_t i = 0; i < v.size(); ++i) PyTuple_SET_ITEM(t, (Py_ssize_t)i, THPVariable_Wrap(v[i]));
  return t;
}

}  // namespace bind
}  // namespace ngl
