// What the parts of the host module share (host_path.cpp, host_operators.cpp): conversions and checks of tensors, the
// library's status as an exception, the refusal of second-order gradients.
#pragma once
#include <torch/extension.h>

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/function.h>

#include <string>

#include "bnb_trunk.h"
#include "host_calls.h"

namespace bnb {
namespace host {

namespace py = pybind11;
using at::Tensor;
using OptTensor = c10::optional<Tensor>;

inline const void* ptr(const OptTensor& t) { return t.has_value() ? t->data_ptr() : nullptr; }

inline Tensor f32c(const Tensor& t) {
  if (t.scalar_type() == at::kBFloat16 && t.is_cuda() && t.is_contiguous() && t.numel() % 8 == 0 &&
      reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0) {
    const c10::cuda::CUDAGuard guard(t.device());
    const Tensor f = at::empty(t.sizes(), t.options().dtype(at::kFloat));
    if (bnb::host::widen(t.data_ptr(), static_cast<float*>(f.data_ptr()), (size_t)t.numel(), at::cuda::getCurrentCUDAStream(t.device().index()).stream()) != BNB_OK)
      throw std::runtime_error("the bfloat16 conversion could not be launched");
    return f;
  }
  const Tensor f = t.scalar_type() == at::kFloat ? t : t.to(at::kFloat);
  return f.is_contiguous() ? f : f.contiguous();
}
inline Tensor contiguous(const Tensor& t) { return t.is_contiguous() ? t : t.contiguous(); }
// One byte per element: a bool tensor as it is, anything else compared with zero.
inline OptTensor bytes_of(const OptTensor& t) {
  if (!t.has_value()) return c10::nullopt;
  return t->scalar_type() == at::kBool ? contiguous(*t) : contiguous(t->ne(0));
}
inline const float* parameter(const Tensor& t, const c10::Device& dev, const char* what) {
  if (t.device() != dev)
    throw std::runtime_error(std::string(what) + " parameter is on " + t.device().str() + ", input on " + dev.str());
  if (t.scalar_type() != at::kFloat || !t.is_contiguous())
    throw std::runtime_error(std::string(what) + " parameter must be contiguous float32 (got " + c10::toString(t.scalar_type()) + ")");
  return static_cast<const float*>(t.data_ptr());
}
inline void check(const char* fn, int status) {
  if (status == BNB_OK) return;
  const std::string text = std::string(fn) + ": " + bnb_status_string(status);
  if (status == BNB_ERR_UNSUPPORTED_DIMS) throw py::value_error(text);
  throw std::runtime_error(text + " (status " + std::to_string(status) + ")");
}
// A bounded wait of an earlier call on this device ran out (its kernels drained and its outputs were
// garbage): say so once, at the next call, without synchronising.
inline void raise_pending_status(const c10::Device& dev) {
  const int st = bnb_last_status();
  if (!st) return;
  bnb_clear_status();
  throw std::runtime_error("an earlier tensor-core call on " + dev.str() + " gave up a bounded wait: " + bnb_status_string(st) +
                           " (status " + std::to_string(st) + "); its outputs, and any state carried from them, are invalid");
}
// Behind the gradients of a backward pass that is itself recorded (create_graph=True): the kernels have no second-order
// gradient, and whoever asks for one is told so, as by an operator without an autograd formula.
struct NoSecondOrder : public torch::autograd::Node {
  torch::autograd::variable_list apply(torch::autograd::variable_list&&) override {
    throw std::runtime_error("the gradients of the CUDA trunk cannot be differentiated again (a second-order gradient through it was asked for)");
  }
};

// The operators outside the trunk (host_operators.cpp) and those behind it in an update (host_update.cpp).
void bind_operators(py::module& m);
void bind_update(py::module& m);

}  // namespace host
}  // namespace bnb
