// What the PyTorch bindings of the operators share: checks, descriptions of tensors, refusals of
// derivatives.  Included by one translation unit.
#pragma once

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/extension.h>

#include <limits>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "causal_conv1d_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Opt = std::optional<Tensor>;

Tensor or_none(const Opt& t) { return t.has_value() ? *t : Tensor(); }
Opt optional_of(const Tensor& t) { return t.defined() ? Opt(t) : std::nullopt; }

std::string shape_text(at::IntArrayRef s) {
  std::string r = "(";
  for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
  return r + (s.size() == 1 ? ",)" : ")");
}

void expect(const char* name, const Tensor& t, at::IntArrayRef shape) {
  if (t.defined() && t.sizes() != shape)
    throw py::value_error(std::string(name) + " must have shape " + shape_text(shape) + ", got " +
                          shape_text(t.sizes()));
}
void expect_dims(const char* name, const Tensor& t, int64_t n) {
  if (t.dim() != n)
    throw py::value_error(std::string(name) + " must have " + std::to_string(n) + " dimensions, got shape " +
                          shape_text(t.sizes()));
}

void one_device(std::initializer_list<const Tensor*> all) {
  const Tensor* first = nullptr;
  for (const Tensor* t : all) {
    if (!t->defined()) continue;
    if (!t->is_cuda()) throw py::value_error("causal_conv1d needs CUDA tensors (there is no CPU implementation)");
    if (!first) first = t;
    else if (t->device() != first->device())
      throw py::value_error("all tensors must be on one device (" + first->device().str() + " vs " +
                            t->device().str() + ")");
  }
}

int32_t dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return CC1D_FLOAT32;
    case at::kHalf: return CC1D_FLOAT16;
    case at::kBFloat16: return CC1D_BFLOAT16;
    case at::kInt: return CC1D_INT32;
    case at::kLong: return CC1D_INT64;
    default: throw py::type_error(std::string("unsupported dtype ") + c10::toString(t));
  }
}

cc1d_tensor describe(const Tensor& t) {
  cc1d_tensor r = {};
  if (!t.defined()) return r;
  r.data = t.data_ptr();
  r.dtype = dtype_code(t.scalar_type());
  for (int64_t i = 0; i < t.dim() && i < 3; ++i) r.stride[i] = t.stride(i);
  return r;
}

void check(int status) {
  if (status == CC1D_OK) return;
  const std::string text = cc1d_last_error();
  switch (status) {
    case CC1D_ERR_VALUE: throw py::value_error(text);
    case CC1D_ERR_TYPE: throw py::type_error(text);
    default: throw std::runtime_error(text.empty() ? "causal_conv1d error" : text);
  }
}

// The current stream of x's device, which is current while this lives.
struct Launch {
  explicit Launch(const Tensor& x)
      : guard(x.device()), stream(c10::cuda::getCurrentCUDAStream(x.get_device()).stream()) {}
  c10::cuda::CUDAGuard guard;
  void* stream;
};

Tensor scratch(int64_t bytes, const Tensor& like) { return at::empty({bytes}, like.options().dtype(at::kByte)); }
Tensor fp32(at::IntArrayRef shape, const Tensor& like) {
  return at::empty(shape, like.options().dtype(at::kFloat));
}

// Refuses forward-mode tangents: a call that dropped one would pass for a function that does not
// depend on that input.
void no_tangents(const char* what, std::initializer_list<const Tensor*> all) {
  for (const Tensor* t : all) {
    if (!t->defined() || !t->_fw_grad(0).defined()) continue;
    py::gil_scoped_acquire gil;
    PyErr_SetString(PyExc_NotImplementedError, (std::string(what) + " has no forward-mode derivative").c_str());
    throw py::error_already_set();
  }
}

// Makes results lead to `inputs` through a node that raises `why` when a derivative is asked for.
void no_derivative(variable_list& results, const variable_list& inputs, const char* why) {
  auto node = std::make_shared<torch::autograd::Error>(why, torch::autograd::collect_next_edges(inputs));
  for (Tensor& r : results)
    if (r.defined()) {
      r = r.detach();
      torch::autograd::set_history(r, node);
    }
}
// The gradients of a node whose backward has no derivative of its own.
variable_list once(variable_list grads, const variable_list& inputs) {
  if (at::GradMode::is_enabled())
    no_derivative(grads, inputs, "trying to differentiate twice a function that was marked with once_differentiable");
  return grads;
}

// t in the layout of ref: a unit stride along the channels or along the sequence.
Tensor like_layout(const Tensor& t, const Tensor& ref) {
  if (!t.defined() || t.dim() != 3 || t.strides() == ref.strides()) return t;
  if (ref.stride(1) == 1 && t.stride(1) != 1) return t.transpose(1, 2).contiguous().transpose(1, 2);
  if (ref.stride(1) != 1 && ref.stride(2) == 1 && t.stride(2) != 1) return t.contiguous();
  return t;
}
Tensor laid_out(const Tensor& x) { return x.stride(1) != 1 && x.stride(2) != 1 ? x.contiguous() : x; }

int64_t state_rows(int64_t batch, const Tensor& seq_idx, std::initializer_list<const Tensor*> states) {
  if (!seq_idx.defined()) return batch;
  for (const Tensor* t : states)
    if (t->defined() && t->dim() > 0) return t->size(0);
  return 0;
}
bool tracked(std::initializer_list<const Tensor*> all) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : all)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// State indices as the C ABI takes them.  What 32 bits do not hold is outside any pool, and has
// to stay so.
Tensor indices32(const Tensor& t) {
  if (!t.defined() || t.scalar_type() == at::kInt) return t;
  switch (t.scalar_type()) {
    case at::kLong: return t.clamp(-1, std::numeric_limits<int32_t>::max()).to(at::kInt);
    case at::kShort:
    case at::kChar:
    case at::kByte: return t.to(at::kInt);
    default: throw py::type_error(std::string("state_indices must be an integer tensor, got ") + c10::toString(t.scalar_type()));
  }
}

}  // namespace
