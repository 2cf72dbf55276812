// What the PyTorch functions share: checks of arguments, layouts, saved tensors, refusals (ops.cpp, train.cpp).
#pragma once
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <ATen/ops/empty.h>
#include <ATen/ops/sub.h>
#include <ATen/ops/zeros.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPException.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>
#include <cmath>
#include <memory>
#include <optional>
#include <sstream>
#include <string>
#include <tuple>
#include <vector>

#include "../../../include/mace_million_amd.h"

namespace {
namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr long kInt32Max = 2147483647L, kMaxRows = 2147483648L - 65536;
constexpr int kMaxDim = 16384, kMaxExperts = 1024, kMaxK = 32, kMaxGroups = 64;

template <typename... A>
std::string text(const A&... a) {
  std::ostringstream s;
  (s << ... << a);
  return s.str();
}

void done(int rc) {
  if (rc != 0) throw std::runtime_error(mm_last_error());
}

mm_stream_t stream() { return (mm_stream_t)c10::hip::getCurrentHIPStream().stream(); }

// Fake, wrapped and zero tensors pass for GPU tensors and have no memory.
void* ptr(const Tensor& t) {
  if (!t.defined()) return nullptr;
  void* p = t.numel() ? t.data_ptr() : nullptr;
  if (!p && t.numel()) throw py::type_error("a tensor without memory (fake, wrapped or zero tensor) cannot be read");
  return p;
}
float* fptr(const Tensor& t) { return (float*)ptr(t); }
int* iptr(const Tensor& t) { return (int*)ptr(t); }

const char* type_name(at::ScalarType t) { return c10::toString(t); }

// dtype code of a floating tensor of the current GPU
int check_gpu(const Tensor& t, const char* name) {
  if (!t.is_cuda()) throw py::type_error(text(name, " must be a GPU tensor"));
  if (t.device().index() != c10::hip::current_device())
    throw py::value_error(text(name, " is on ", t.device(), ", the current device is cuda:",
                               (int)c10::hip::current_device()));
  switch (t.scalar_type()) {
    case at::kFloat: return 0;
    case at::kBFloat16: return 1;
    case at::kHalf: return 2;
    default:
      throw py::type_error(text(name, " must be float32, bfloat16 or float16, got ", type_name(t.scalar_type())));
  }
}

Tensor f32(at::IntArrayRef size, const Tensor& like) { return at::empty(size, like.options().dtype(at::kFloat)); }
Tensor i32(at::IntArrayRef size, const Tensor& like) { return at::empty(size, like.options().dtype(at::kInt)); }

// The values of a lazily negated view (of a conjugate's imaginary part, say) are not those of its memory.
Tensor plain(const Tensor& t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }

// Autograd takes absent tensors as empty optionals.
using Maybe = std::optional<Tensor>;
Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); }
Tensor value(const Maybe& t) { return t ? *t : Tensor(); }

bool needs_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// Forward-mode derivatives and traces go through dispatched operations only, so they would miss these functions without
// a word: the result would pass for a constant, the trace would hold memory that nothing writes.
void refuse_modes(const char* what, std::initializer_list<const Tensor*> ts) {
  if (torch::jit::tracer::isTracing()) throw std::runtime_error(text(what, " cannot be traced (torch.jit.trace)"));
  for (const Tensor* t : ts)
    if (t->defined() && t->_fw_grad(0).defined())
      throw std::runtime_error(text(what, " has no forward-mode derivative: its inputs must not be dual tensors"));
}

// Gradients that raise when they are differentiated again, instead of passing for constants.
variable_list once(variable_list grads, const char* what) {
  if (!at::GradMode::is_enabled()) return grads;
  for (Tensor& g : grads)
    if (g.defined()) g = g.detach().requires_grad_(true);
  auto error = std::make_shared<torch::autograd::DelayedError>(text(what, " can be differentiated once only"),
                                                               (int64_t)grads.size());
  return (*error)(std::move(grads));
}

// t as rows with a contiguous last axis, and the distance of rows
std::pair<Tensor, long> as_rows(Tensor t) {
  const long D = t.size(-1);
  if (t.dim() != 2) t = t.reshape({-1, D});
  if (D > 1 && t.stride(1) != 1) t = t.contiguous();
  return {t, t.size(0) > 1 ? t.stride(0) : D};
}

// A saved tensor as its node gets it back.  Hooks on saved tensors (offloading, compression) may return it with any
// strides, so its layout is taken from what comes back; sizes and type have to be those that were saved.
Tensor unpacked(const Tensor& t, at::IntArrayRef size, at::ScalarType type, const Tensor& like,
                       const char* name) {
  if (t.defined() && (t.sizes() != size || t.scalar_type() != type || t.device() != like.device()))
    throw std::runtime_error(text(name, " was saved for the backward as ", type_name(type), " ", size, " on ",
                                  like.device(), " and came back as ", type_name(t.scalar_type()), " ", t.sizes(),
                                  " on ", t.device()));
  return plain(t);
}

Tensor unpacked_dense(const Tensor& t, at::IntArrayRef size, at::ScalarType type, const Tensor& like,
                      const char* name) {
  const Tensor u = unpacked(t, size, type, like, name);
  return u.defined() ? u.contiguous() : u;
}

at::ScalarType type_of(int64_t code) { return code == 0 ? at::kFloat : code == 1 ? at::kBFloat16 : at::kHalf; }
}  // namespace

void bind_train(py::module_& m);   // train.cpp
