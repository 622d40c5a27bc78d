// What the operators' entry points on torch tensors share (policy_torch.cpp, policy_memory_torch.cpp): argument checks, rows,
// streams, autograd's odds and ends.  Each file has its own copy of everything here.
#pragma once
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include "isaac_net_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

PyObject* unsupported = nullptr;      // engine.B200Unsupported

// ------------------------------------------------------------------------------------------------- checks
// Messages are put together by hand: formatting a shape through torch's own operator<< crashed in libraries built here
// against the installed torch (a three-line extension shows it).
std::string text(const char* v) { return v; }
std::string text(const std::string& v) { return v; }
std::string text(int64_t v) { return std::to_string(v); }
std::string text(double v) { return std::to_string(v); }
std::string text(at::ScalarType v) { return c10::toString(v); }
std::string text(at::IntArrayRef v) {
  std::string s = "[";
  for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + std::to_string(v[i]);
  return s + "]";
}
template <typename... A>
std::string join(const A&... a) {
  std::string s;
  ((s += text(a)), ...);
  return s;
}
// What the checks raise; called from Python only
template <typename... A>
[[noreturn]] void refuse(const A&... a) {
  PyErr_SetString(unsupported, join(a...).c_str());
  throw py::error_already_set();
}
#define VALUE_CHECK(ok, ...) \
  if (!(ok)) throw py::value_error(join(__VA_ARGS__))

int type_code(at::ScalarType t) {
  return t == at::kBFloat16 ? INB_BF16 : t == at::kHalf ? INB_F16 : t == at::kFloat ? INB_F32 : -1;
}
void on_cuda(const Tensor& t, const char* name) {
  if (!t.is_cuda()) refuse(name, " is on ", t.device().str(), ": the policy operators run on CUDA tensors only");
}
// An operator's first tensor: on a CUDA device, of one of the operators' types
int first(const Tensor& x, const char* name, bool fp32 = true) {
  const int code = type_code(x.scalar_type());
  on_cuda(x, name);
  if (code < 0 || (code == INB_F32 && !fp32))
    refuse(name, " is ", x.scalar_type(), ": this operator takes bfloat16", fp32 ? ", float16 and float32" : " and float16");
  return code;
}
void same(const Tensor& t, const char* name, const Tensor& like, at::ScalarType want) {
  if (t.is_cuda() && t.get_device() == like.get_device() && t.scalar_type() == want) return;
  on_cuda(t, name);
  VALUE_CHECK(t.device() == like.device(), name, " is on ", t.device().str(), ", the first tensor on ", like.device().str());
  throw py::type_error(join(name, " is ", t.scalar_type(), ", expected ", want));
}
void vector(const Tensor& t, const char* name, int64_t n) {
  VALUE_CHECK(t.dim() == 1 && t.size(0) == n, name, " must have shape [", n, "], got ", t.sizes());
}
int64_t width(const Tensor& x, const char* name) {
  VALUE_CHECK(x.dim() >= 1 && x.size(-1) >= 1, name, " must be [..., D] with D >= 1, got shape ", x.sizes());
  return x.size(-1);
}

// [..., D] as rows of one stride; a copy where there is none, or where elements are not contiguous
struct Rows {
  Tensor t;
  int64_t ld = 0;
  const void* p() const { return t.defined() ? t.const_data_ptr() : nullptr; }
};
Rows rows_of(const Tensor& t, int64_t d, int64_t most = INT64_MAX) {
  if (!t.defined()) return {};
  if (t.is_contiguous()) return {t, d};
  bool one = t.stride(-1) == 1 || d == 1;
  int64_t ld = -1, next = 0;      // the rows' stride, and the stride that the next axis out has to have
  for (int64_t i = t.dim() - 2; one && i >= 0; --i) {
    if (t.size(i) == 1) continue;
    if (ld < 0)
      ld = t.stride(i);
    else
      one = t.stride(i) == next;
    next = t.stride(i) * t.size(i);
  }
  if (one && ld <= most) return {t, ld < 0 ? d : ld};
  return {t.contiguous(), d};
}
const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* out(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
Tensor like(const Tensor& t) { return t.defined() ? at::empty(t.sizes(), t.options()) : Tensor(); }

// The current stream of a tensor's device, which is the current device while this lives
struct On {
  c10::cuda::CUDAGuard guard;
  void* stream;
  explicit On(const Tensor& t) : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.get_device()).stream()) {}
};
void check(int rc, const char* name) {
  if (rc != 0) throw std::runtime_error(join(name, " failed with status ", (int64_t)rc));
}

bool any_grad(std::initializer_list<Tensor> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor& t : ts)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}
// Forward-mode derivatives are not there: a tangent that came in would be lost, which reads as a zero derivative
void no_tangents(std::initializer_list<std::pair<const Tensor*, const char*>> ts) {
  for (const auto& [t, name] : ts)
    if (t != nullptr && t->_fw_grad(/*level=*/0).defined())
      refuse(name, " carries a tangent: the policy operators have no forward-mode derivatives");
}
const Tensor* given(const std::optional<Tensor>& t) { return t ? &*t : nullptr; }
// A backward pass's results, which cannot be differentiated again: an attempt raises
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  for (Tensor& g : grads)
    if (g.defined()) g = g.detach().requires_grad_(true);
  auto stop = std::make_shared<torch::autograd::DelayedError>("the policy operators can be differentiated once only",
                                                              (int64_t)grads.size());
  return (*stop)(std::move(grads));
}

}  // namespace
