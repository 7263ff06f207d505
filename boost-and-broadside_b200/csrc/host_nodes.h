// What the host sides of the operators beside the trunk share (host_operators.cpp, host_update.cpp): checks of arguments, tensors as
// the kernels read them, the autograd node of an eager call.
#pragma once
#include "host_tensors.h"

#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>

#include <functional>
#include <sstream>
#include <string>
#include <utility>
#include <vector>

namespace bnb {
namespace host {

using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

[[noreturn]] inline void refuse(const std::string& text) { throw std::runtime_error(text); }
inline std::string shape_text(at::IntArrayRef s) {
  std::ostringstream o;
  o << "(";
  for (size_t i = 0; i < s.size(); ++i) o << (i ? ", " : "") << s[i];
  o << (s.size() == 1 ? ",)" : ")");
  return o.str();
}
inline OptTensor given(const OptTensor& t) { return t.has_value() && t->defined() ? t : c10::nullopt; }
inline OptTensor opt(const Tensor& t) { return t.defined() ? OptTensor(t) : c10::nullopt; }

inline int element_of(const char* fn, const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return BNB_ELEM_F32;
    case at::kBFloat16: return BNB_ELEM_BF16;
    case at::kHalf: return BNB_ELEM_F16;
    default: throw py::value_error(std::string(fn) + ": inputs must be float32, bfloat16 or float16, got " + c10::toString(t.scalar_type()));
  }
}
inline void expect(const char* fn, const char* name, const Tensor& t, at::IntArrayRef sizes, const c10::Device& dev) {
  if (t.sizes() != sizes) refuse(std::string(fn) + ": " + name + " must have shape " + shape_text(sizes) + ", got " + shape_text(t.sizes()));
  if (t.device() != dev) refuse(std::string(fn) + ": " + name + " is on " + t.device().str() + ", the input on " + dev.str());
}
inline void expect_type(const char* fn, const char* name, const Tensor& t, at::ScalarType type) {
  if (t.scalar_type() != type)
    refuse(std::string(fn) + ": " + name + " must be " + c10::toString(type) + ", got " + c10::toString(t.scalar_type()));
}
inline void expect_cuda(const char* fn, const Tensor& t) {
  if (!t.is_cuda()) refuse(std::string(fn) + ": the input is on " + t.device().str() + "; the kernels run on CUDA only (sm_100a) and have no CPU path");
}
// A float32 parameter or state as the kernels read it: contiguous, on a 16-byte boundary.  A copy is put into `held` until the call is
// queued.
inline const float* floats(const Tensor& t, std::vector<Tensor>& held) {
  Tensor v = t.is_contiguous() ? t : t.contiguous();
  if (reinterpret_cast<uintptr_t>(v.data_ptr()) % 16) v = v.clone();
  held.push_back(v);
  return static_cast<const float*>(v.data_ptr());
}
inline const float* floats(const OptTensor& t, std::vector<Tensor>& held) { return t.has_value() ? floats(*t, held) : nullptr; }
template <class P> P* data(const OptTensor& t) { return t.has_value() ? static_cast<P*>(t->data_ptr()) : nullptr; }
inline void* stream_of(const c10::Device& dev) { return at::cuda::getCurrentCUDAStream(dev.index()).stream(); }
inline Tensor scratch_of(size_t bytes, const Tensor& like) { return at::empty({(int64_t)std::max<size_t>(bytes, 16)}, like.options().dtype(at::kByte)); }
inline int fits_int(const char* fn, int64_t v) {
  if (v > INT32_MAX) throw py::value_error(std::string(fn) + ": a dimension above 2^31 - 1");
  return (int)v;
}
// The autograd node of an eager call: saved inputs (and what the forward kept), and the backward as a function of them.
struct OpNode : public torch::autograd::Node {
  using Backward = std::function<variable_list(const std::vector<Tensor>&, const variable_list&)>;
  std::vector<SavedVariable> saved;
  Backward backward;
  size_t inputs = 0;   // the first of `saved` that are differentiable inputs, for the edges of a recorded backward

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    const bool recorded = at::GradMode::is_enabled();
    const at::NoGradGuard no_grad;
    std::vector<Tensor> in;
    in.reserve(saved.size());
    for (auto& s : saved) in.push_back(s.unpack());
    variable_list out = backward(in, grads);
    for (size_t i = 0; i < out.size(); ++i)
      if (!task_should_compute_output(i)) out[i] = Tensor();
    if (recorded) {
      variable_list from(in.begin(), in.begin() + inputs);
      from.insert(from.end(), grads.begin(), grads.end());
      auto again = std::make_shared<NoSecondOrder>();
      again->set_next_edges(torch::autograd::collect_next_edges(from));
      for (Tensor& t : out)
        if (t.defined()) {
          t = t.detach();
          torch::autograd::create_gradient_edge(t, again);
        }
    }
    return out;
  }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (auto& s : saved) s.reset_data();
  }
};
inline bool wants_grad(const variable_list& inputs) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor& t : inputs)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}
inline std::shared_ptr<OpNode> node_of(const variable_list& inputs, const variable_list& others, OpNode::Backward backward) {
  auto node = std::make_shared<OpNode>();
  node->set_next_edges(torch::autograd::collect_next_edges(inputs));
  node->inputs = inputs.size();
  for (const Tensor& t : inputs) node->saved.emplace_back(t, false);
  for (const Tensor& t : others) node->saved.emplace_back(t, false);
  node->backward = std::move(backward);
  return node;
}
inline Tensor value(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }

// x as (rows, width), its rows contiguous elements.
inline Tensor rows_of(const Tensor& t) {
  const Tensor v = t.reshape({-1, t.size(-1)});
  return v.stride(1) == 1 || v.size(1) <= 1 ? v : v.contiguous();
}
inline int64_t row_stride(const Tensor& v) { return v.size(0) > 1 ? v.stride(0) : v.size(1); }

}  // namespace host
}  // namespace bnb
