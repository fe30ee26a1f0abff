// autograd_common.h -- what the autograd nodes of the operators share (host
// code only).
#ifndef AUTOGRAD_COMMON_H_
#define AUTOGRAD_COMMON_H_

#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>

#include <stdexcept>
#include <string>

#include "dsx.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// A status other than 0: the library's message as a RuntimeError.
void check_status(const char* name, int rc, const char* (*last_error)()) {
  if (rc) throw std::runtime_error(std::string(name) + " failed (status " + std::to_string(rc) + "): " + last_error());
}

// The library's kernels see values alone: a forward-mode tangent of an input
// would be lost on the way to the output, which reads as a tangent of zero.
void refuse_tangent(const char* name, const Tensor& t) {
  if (t.defined() && t._fw_grad(0).defined())
    throw std::runtime_error(std::string(name) + " has no forward-mode derivative: an input carries a tangent");
}

int32_t code_of(at::ScalarType t) { return t == at::kFloat ? DSX_F32 : t == at::kHalf ? DSX_F16 : DSX_BF16; }

// t [n, d], or a copy where its columns are not adjacent or its rows overlap.
Tensor rows_of(const Tensor& t) {
  if (!t.defined() || t.is_contiguous()) return t;
  const int64_t n = t.size(0), d = t.size(1);
  if ((d > 1 && t.stride(1) != 1) || (n > 1 && t.stride(0) < d)) return t.contiguous();
  return t;
}
int64_t ld_of(const Tensor& t) { return !t.defined() ? 0 : t.size(0) > 1 ? t.stride(0) : t.size(1); }
void* at_of(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// `bytes` as the library's size functions return them: below 0 is a refusal.
Tensor scratch_of(int64_t bytes, const Tensor& like, const char* (*last_error)()) {
  if (bytes < 0) throw std::runtime_error(last_error());
  return at::empty({bytes}, like.options().dtype(at::kByte).requires_grad(false));
}
Tensor result(const Tensor& like) { return at::empty(like.sizes(), like.options().requires_grad(false)); }

// Results of a backward that was asked to be differentiable again: an error
// when that is tried, as torch's once_differentiable has it.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list defined;
  for (auto& g : grads)
    if (g.defined()) defined.push_back(g.detach().requires_grad_(true));
  const int count = static_cast<int>(defined.size());
  auto node = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that is differentiable once", count);
  variable_list marked = (*node)(std::move(defined));
  size_t k = 0;
  for (auto& g : grads)
    if (g.defined()) g = marked[k++];
  return grads;
}

template <class F>
void bind_one(F& f, const pybind11::dict& d, const char* name) {
  f = reinterpret_cast<F>(d[name].cast<uintptr_t>());
}

}  // namespace

#endif  // AUTOGRAD_COMMON_H_
