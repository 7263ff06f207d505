// The host side of the operators outside the trunk (yemong/selective.py, yemong/gated.py): checks, outputs from torch's
// allocator, the launch, and the autograd nodes of eager calls.  Scratch comes from torch's allocator call by call, so that
// captured graphs and streams never share any.
#include "host_tensors.h"

#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>

#include <functional>
#include <sstream>
#include <tuple>
#include <vector>

namespace bnb {
namespace host {
namespace {

using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

[[noreturn]] void refuse(const std::string& text) { throw std::runtime_error(text); }
std::string shape_text(at::IntArrayRef s) {
  std::ostringstream o;
  o << "(";
  for (size_t i = 0; i < s.size(); ++i) o << (i ? ", " : "") << s[i];
  o << (s.size() == 1 ? ",)" : ")");
  return o.str();
}
OptTensor given(const OptTensor& t) { return t.has_value() && t->defined() ? t : c10::nullopt; }
OptTensor opt(const Tensor& t) { return t.defined() ? OptTensor(t) : c10::nullopt; }

int element_of(const char* fn, const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return BNB_ELEM_F32;
    case at::kBFloat16: return BNB_ELEM_BF16;
    case at::kHalf: return BNB_ELEM_F16;
    default: throw py::value_error(std::string(fn) + ": inputs must be float32, bfloat16 or float16, got " + c10::toString(t.scalar_type()));
  }
}
void expect(const char* fn, const char* name, const Tensor& t, at::IntArrayRef sizes, const c10::Device& dev) {
  if (t.sizes() != sizes) refuse(std::string(fn) + ": " + name + " must have shape " + shape_text(sizes) + ", got " + shape_text(t.sizes()));
  if (t.device() != dev) refuse(std::string(fn) + ": " + name + " is on " + t.device().str() + ", the input on " + dev.str());
}
void expect_type(const char* fn, const char* name, const Tensor& t, at::ScalarType type) {
  if (t.scalar_type() != type)
    refuse(std::string(fn) + ": " + name + " must be " + c10::toString(type) + ", got " + c10::toString(t.scalar_type()));
}
void expect_cuda(const char* fn, const Tensor& t) {
  if (!t.is_cuda()) refuse(std::string(fn) + ": the input is on " + t.device().str() + "; the kernels run on CUDA only (sm_100a) and have no CPU path");
}
// A float32 parameter or state as the kernels read it: contiguous, on a 16-byte boundary.  A copy is put into `held` until the call is
// queued.
const float* floats(const Tensor& t, std::vector<Tensor>& held) {
  Tensor v = t.is_contiguous() ? t : t.contiguous();
  if (reinterpret_cast<uintptr_t>(v.data_ptr()) % 16) v = v.clone();
  held.push_back(v);
  return static_cast<const float*>(v.data_ptr());
}
const float* floats(const OptTensor& t, std::vector<Tensor>& held) { return t.has_value() ? floats(*t, held) : nullptr; }
// (T, R, ...) with unit innermost stride.
BnbView view_of(const Tensor& t, std::vector<Tensor>& held) {
  const Tensor v = t.stride(-1) == 1 || t.size(-1) <= 1 ? t : t.contiguous();
  held.push_back(v);
  const bool stepped = v.dim() >= 3;
  BnbView o{};
  o.data = v.data_ptr();
  o.step = stepped ? v.stride(0) : 0;
  o.row = v.stride(stepped ? 1 : 0);
  return o;
}
// (.., G, N): groups in the last but one dimension.
BnbView shared_view(const Tensor& t, std::vector<Tensor>& held) {
  const Tensor v = t.stride(-1) == 1 || t.size(-1) <= 1 ? t : t.contiguous();
  held.push_back(v);
  const bool stepped = v.dim() == 4;
  BnbView o{};
  o.data = v.data_ptr();
  o.step = stepped ? v.stride(0) : 0;
  o.row = v.stride(stepped ? 1 : 0);
  o.group = v.stride(-2);
  return o;
}
// A new dense tensor of x's shape that lies in memory as x does: step by step, or row by row (batch-major programs).  It is no view
// of another: a differentiated call's result could not be changed in place then.
Tensor rows_like(const Tensor& x) {
  if (x.dim() < 3 || x.stride(0) >= x.stride(1)) return at::empty(x.sizes(), x.options());
  return at::empty_strided(x.sizes(), {x.size(2), x.size(0) * x.size(2), 1}, x.options());
}
OptTensor done_bytes(const char* fn, const OptTensor& done, int64_t T, int64_t R, const c10::Device& dev) {
  if (!done.has_value()) return c10::nullopt;
  expect(fn, "done", *done, {T, R}, dev);
  return bytes_of(done);
}
// As the kernels read them, which clamp to 0 .. T themselves: values of 64 bits are clamped before they lose their upper half.
OptTensor row_lengths(const char* fn, const OptTensor& lengths, int64_t T, int64_t R, const c10::Device& dev) {
  if (!lengths.has_value()) return c10::nullopt;
  expect(fn, "lengths", *lengths, {R}, dev);
  if (lengths->scalar_type() != at::kInt && lengths->scalar_type() != at::kLong) refuse(std::string(fn) + ": lengths must be int32 or int64");
  return contiguous(lengths->scalar_type() == at::kLong ? lengths->clamp(0, T).to(at::kInt) : *lengths);
}
OptTensor reset_bytes(const char* fn, const OptTensor& reset, int64_t R, const c10::Device& dev) {
  if (!reset.has_value()) return c10::nullopt;
  expect(fn, "reset", *reset, {R}, dev);
  return bytes_of(reset);
}
template <class P> P* data(const OptTensor& t) { return t.has_value() ? static_cast<P*>(t->data_ptr()) : nullptr; }
void* stream_of(const c10::Device& dev) { return at::cuda::getCurrentCUDAStream(dev.index()).stream(); }
Tensor scratch_of(size_t bytes, const Tensor& like) { return at::empty({(int64_t)std::max<size_t>(bytes, 16)}, like.options().dtype(at::kByte)); }
int fits_int(const char* fn, int64_t v) {
  if (v > INT32_MAX) throw py::value_error(std::string(fn) + ": a dimension above 2^31 - 1");
  return (int)v;
}
// A state that a step updates in place.
void expect_state(const char* fn, const Tensor& s, at::IntArrayRef sizes, const c10::Device& dev) {
  expect(fn, "state", s, sizes, dev);
  expect_type(fn, "state", s, at::kFloat);
  if (!s.is_contiguous() || reinterpret_cast<uintptr_t>(s.data_ptr()) % 16)
    refuse(std::string(fn) + ": the state is updated in place and must be contiguous, on a 16-byte boundary");
  if (s.is_inference() && !c10::InferenceMode::is_enabled())   // as autograd does, but before the kernel has run
    refuse(std::string(fn) + ": the state is updated in place and was made in inference mode, outside of which it must not be changed");
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
bool wants_grad(const variable_list& inputs) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor& t : inputs)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}
std::shared_ptr<OpNode> node_of(const variable_list& inputs, const variable_list& others, OpNode::Backward backward) {
  auto node = std::make_shared<OpNode>();
  node->set_next_edges(torch::autograd::collect_next_edges(inputs));
  node->inputs = inputs.size();
  for (const Tensor& t : inputs) node->saved.emplace_back(t, false);
  for (const Tensor& t : others) node->saved.emplace_back(t, false);
  node->backward = std::move(backward);
  return node;
}
Tensor value(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }

// ------------------------------------------------------------------ causal convolution

struct ConvCall {
  BnbCausalConv c{};
  std::vector<Tensor> held;
  OptTensor done, lengths;
};
ConvCall conv_call(const char* fn, const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& state, const OptTensor& done,
                   const OptTensor& lengths, int activation) {
  expect_cuda(fn, x);
  if (x.dim() != 3) refuse(std::string(fn) + ": x must have shape (T, R, C), got " + shape_text(x.sizes()));
  const int64_t T = x.size(0), R = x.size(1), C = x.size(2);
  const c10::Device dev = x.device();
  ConvCall k;
  BnbCausalConv& c = k.c;
  c.element = element_of(fn, x);
  if (weight.dim() != 2) refuse(std::string(fn) + ": weight must have shape (" + std::to_string(C) + ", taps), got " + shape_text(weight.sizes()));
  const int64_t K = weight.size(1);
  if (K < 2 || K > 4) throw py::value_error(std::string(fn) + ": 2 to 4 taps are built, got " + std::to_string(K));
  expect(fn, "weight", weight, {C, K}, dev);
  expect_type(fn, "weight", weight, at::kFloat);
  if (bias.has_value()) {
    expect(fn, "bias", *bias, {C}, dev);
    expect_type(fn, "bias", *bias, at::kFloat);
  }
  if (state.has_value()) {
    expect(fn, "state", *state, {R, K - 1, C}, dev);
    expect_type(fn, "state", *state, at::kFloat);
  }
  k.done = done_bytes(fn, done, T, R, dev);
  k.lengths = row_lengths(fn, lengths, T, R, dev);
  c.steps = fits_int(fn, T);
  c.rows = fits_int(fn, R);
  c.width = fits_int(fn, C);
  c.taps = (int)K;
  c.activation = activation;
  c.x = view_of(x, k.held);
  c.weight = floats(weight, k.held);
  c.bias = floats(bias, k.held);
  c.state_in = floats(state, k.held);
  c.done = data<uint8_t>(k.done);
  c.lengths = data<int32_t>(k.lengths);
  return k;
}

std::tuple<Tensor, Tensor> conv_forward(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& state, const OptTensor& done,
                                        const OptTensor& lengths, int activation) {
  const c10::cuda::OptionalCUDAGuard guard(x.is_cuda() ? c10::optional<c10::Device>(x.device()) : c10::nullopt);
  ConvCall k = conv_call("causal_conv", x, weight, bias, state, done, lengths, activation);
  const Tensor y = rows_like(x), out = at::empty({x.size(1), weight.size(1) - 1, x.size(2)}, weight.options());
  k.c.y = view_of(y, k.held);
  k.c.state_out = static_cast<float*>(out.data_ptr());
  check("bnb_causal_conv_fwd", bnb_causal_conv_fwd(&k.c, stream_of(x.device())));
  return {y, out};
}

// Gradients of x, weight, bias and state for dy and dstate (either may be missing).
std::vector<Tensor> conv_backward(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& state, const OptTensor& done,
                                  const OptTensor& lengths, int activation, const OptTensor& dy, const OptTensor& dstate) {
  const c10::cuda::CUDAGuard guard(x.device());
  ConvCall k = conv_call("causal_conv", x, weight, bias, state, done, lengths, activation);
  BnbCausalConvGrads g{};
  const Tensor gy = dy.has_value() ? dy->to(x.scalar_type()) : at::zeros_like(x);
  expect("causal_conv", "the gradient of y", gy, x.sizes(), x.device());
  const Tensor dx = rows_like(x), dw = at::empty_like(weight, at::MemoryFormat::Contiguous);
  const Tensor db = bias.has_value() ? at::empty({x.size(2)}, weight.options()) : Tensor();
  const Tensor ds = state.has_value() ? at::empty(state->sizes(), state->options()) : Tensor();
  g.dy = view_of(gy, k.held);
  g.dx = view_of(dx, k.held);
  g.dstate_out = floats(dstate, k.held);
  g.dstate_in = ds.defined() ? static_cast<float*>(ds.data_ptr()) : nullptr;
  g.dweight = static_cast<float*>(dw.data_ptr());
  g.dbias = db.defined() ? static_cast<float*>(db.data_ptr()) : nullptr;
  const Tensor scratch = scratch_of(bnb_causal_conv_bwd_scratch_bytes(&k.c), x);
  check("bnb_causal_conv_bwd", bnb_causal_conv_bwd(&k.c, &g, scratch.data_ptr(), (size_t)scratch.numel(), stream_of(x.device())));
  return {dx, dw, db, ds};
}

std::tuple<Tensor, Tensor> conv(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& state, const OptTensor& done,
                                const OptTensor& lengths, int activation) {
  const variable_list inputs{x, weight, value(bias), value(state)};
  if (!wants_grad(inputs)) return conv_forward(x, weight, bias, state, done, lengths, activation);
  auto node = node_of(inputs, {value(done), value(lengths)}, [activation](const std::vector<Tensor>& s, const variable_list& g) -> variable_list {
    return conv_backward(s[0], s[1], opt(s[2]), opt(s[3]), opt(s[4]), opt(s[5]), activation, opt(g[0]), opt(g[1]));
  });
  Tensor y, out;
  {
    const at::NoGradGuard no_grad;
    std::tie(y, out) = conv_forward(x, weight, bias, state, done, lengths, activation);
  }
  torch::autograd::create_gradient_edge(y, node);
  torch::autograd::create_gradient_edge(out, node);
  return {y, out};
}

Tensor conv_step(const Tensor& x, const Tensor& state, const Tensor& weight, const OptTensor& bias, const OptTensor& reset, int activation) {
  const char* fn = "causal_conv_step";
  expect_cuda(fn, x);
  if (x.dim() != 2) refuse(std::string(fn) + ": x must have shape (R, C), got " + shape_text(x.sizes()));
  const c10::cuda::CUDAGuard guard(x.device());
  ConvCall k = conv_call(fn, x.unsqueeze(0), weight, bias, c10::nullopt, c10::nullopt, c10::nullopt, activation);
  expect_state(fn, state, {x.size(0), weight.size(1) - 1, x.size(1)}, x.device());
  const OptTensor cleared = reset_bytes(fn, reset, x.size(0), x.device());
  const Tensor y = at::empty(x.sizes(), x.options());
  k.c.y = view_of(y, k.held);
  k.c.state_out = static_cast<float*>(state.data_ptr());
  k.c.state_in = k.c.state_out;
  k.c.reset = data<uint8_t>(cleared);
  check("bnb_causal_conv_fwd", bnb_causal_conv_fwd(&k.c, stream_of(x.device())));
  state.unsafeGetTensorImpl()->bump_version();
  return y;
}

// ------------------------------------------------------------------ selective scan

struct ScanCall {
  BnbSelectiveScan q{};
  std::vector<Tensor> held;
  OptTensor done, lengths;
};
// u, delta, z (T, R, C) or (R, C); b, c the same with (G, N) in the place of C.
ScanCall scan_call(const char* fn, const Tensor& u, const Tensor& delta, const Tensor& a, const Tensor& b, const Tensor& c, const OptTensor& d, const OptTensor& z,
                   const OptTensor& bias, bool softplus) {
  expect_cuda(fn, u);
  const bool stepped = u.dim() == 3;
  const c10::Device dev = u.device();
  const int64_t C = u.size(-1), R = u.size(stepped ? 1 : 0), T = stepped ? u.size(0) : 1;
  ScanCall k;
  BnbSelectiveScan& q = k.q;
  q.element = element_of(fn, u);
  if (a.dim() != 2) refuse(std::string(fn) + ": A must have shape (" + std::to_string(C) + ", N), got " + shape_text(a.sizes()));
  const int64_t N = a.size(1);
  if (N < 1 || N > 64) throw py::value_error(std::string(fn) + ": 1 to 64 states a channel are built, got " + std::to_string(N));
  expect(fn, "A", a, {C, N}, dev);
  expect_type(fn, "A", a, at::kFloat);
  if (b.dim() != u.dim() + 1) refuse(std::string(fn) + ": B must have shape (.., groups, N), got " + shape_text(b.sizes()));
  const int64_t G = b.size(-2);
  if (G < 1 || C % G) throw py::value_error(std::string(fn) + ": the groups of B and C must divide the width " + std::to_string(C) + ", got " + std::to_string(G));
  std::vector<int64_t> shared = u.sizes().vec();
  shared.back() = G;
  shared.push_back(N);
  expect(fn, "delta", delta, u.sizes(), dev);
  expect(fn, "B", b, shared, dev);
  expect(fn, "C", c, shared, dev);
  for (const auto& [name, t] : {std::pair<const char*, const Tensor*>{"delta", &delta}, {"B", &b}, {"C", &c}}) expect_type(fn, name, *t, u.scalar_type());
  if (z.has_value()) {
    expect(fn, "z", *z, u.sizes(), dev);
    expect_type(fn, "z", *z, u.scalar_type());
    q.z = view_of(*z, k.held);
  }
  for (const auto& [name, t] : {std::pair<const char*, const OptTensor*>{"D", &d}, {"delta_bias", &bias}})
    if (t->has_value()) {
      expect(fn, name, **t, {C}, dev);
      expect_type(fn, name, **t, at::kFloat);
    }
  q.steps = fits_int(fn, T);
  q.rows = fits_int(fn, R);
  q.width = fits_int(fn, C);
  q.states = (int)N;
  q.groups = (int)G;
  q.softplus = softplus ? 1 : 0;
  q.u = view_of(u, k.held);
  q.delta = view_of(delta, k.held);
  q.b = shared_view(b, k.held);
  q.c = shared_view(c, k.held);
  q.a = floats(a, k.held);
  q.d = floats(d, k.held);
  q.delta_bias = floats(bias, k.held);
  return k;
}
ScanCall scan_sequence(const Tensor& u, const Tensor& delta, const Tensor& a, const Tensor& b, const Tensor& c, const OptTensor& d, const OptTensor& z,
                       const OptTensor& bias, const OptTensor& state, const OptTensor& done, const OptTensor& lengths, bool softplus) {
  const char* fn = "selective_scan";
  if (u.dim() != 3) refuse(std::string(fn) + ": u must have shape (T, R, C), got " + shape_text(u.sizes()));
  ScanCall k = scan_call(fn, u, delta, a, b, c, d, z, bias, softplus);
  if (state.has_value()) {
    expect(fn, "state", *state, {u.size(1), u.size(2), a.size(1)}, u.device());
    expect_type(fn, "state", *state, at::kFloat);
    k.q.state_in = floats(*state, k.held);
  }
  k.done = done_bytes(fn, done, u.size(0), u.size(1), u.device());
  k.lengths = row_lengths(fn, lengths, u.size(0), u.size(1), u.device());
  k.q.done = data<uint8_t>(k.done);
  k.q.lengths = data<int32_t>(k.lengths);
  return k;
}

// (y, state behind the last step, states kept for the backward: empty unless asked for)
std::tuple<Tensor, Tensor, Tensor> scan_forward(const Tensor& u, const Tensor& delta, const Tensor& a, const Tensor& b, const Tensor& c, const OptTensor& d,
                                                const OptTensor& z, const OptTensor& bias, const OptTensor& state, const OptTensor& done,
                                                const OptTensor& lengths, bool softplus, bool keep) {
  const c10::cuda::OptionalCUDAGuard guard(u.is_cuda() ? c10::optional<c10::Device>(u.device()) : c10::nullopt);
  ScanCall k = scan_sequence(u, delta, a, b, c, d, z, bias, state, done, lengths, softplus);
  const Tensor y = rows_like(u), out = at::empty({u.size(1), u.size(2), a.size(1)}, a.options());
  k.q.y = view_of(y, k.held);
  k.q.state_out = static_cast<float*>(out.data_ptr());
  const Tensor kept = at::empty({keep ? (int64_t)(bnb_selective_scan_kept_bytes(&k.q) / 4) : 0}, a.options());
  if (keep) k.q.kept = static_cast<float*>(kept.data_ptr());
  const size_t bytes = bnb_selective_scan_scratch_bytes(&k.q);
  const Tensor scratch = bytes ? scratch_of(bytes, u) : Tensor();
  check("bnb_selective_scan_fwd", bnb_selective_scan_fwd(&k.q, bytes ? scratch.data_ptr() : nullptr, bytes, stream_of(u.device())));
  return {y, out, kept};
}

// Gradients of u, delta, A, B, C, D, z, delta_bias and state.
std::vector<Tensor> scan_backward(const Tensor& u, const Tensor& delta, const Tensor& a, const Tensor& b, const Tensor& c, const OptTensor& d, const OptTensor& z,
                                  const OptTensor& bias, const OptTensor& state, const OptTensor& done, const OptTensor& lengths, bool softplus,
                                  const Tensor& kept, const OptTensor& dy, const OptTensor& dstate) {
  const c10::cuda::CUDAGuard guard(u.device());
  ScanCall k = scan_sequence(u, delta, a, b, c, d, z, bias, state, done, lengths, softplus);
  const Tensor states = contiguous(kept).to(u.device());
  if (states.scalar_type() != at::kFloat || (size_t)states.numel() * 4 != bnb_selective_scan_kept_bytes(&k.q))
    refuse("selective_scan: the kept states came back as another tensor: saved-tensor hooks have to return type and shape as they were");
  std::vector<Tensor>& held = k.held;
  k.q.kept = const_cast<float*>(floats(states, held));
  BnbSelectiveScanGrads g{};
  const Tensor gy = dy.has_value() ? dy->to(u.scalar_type()) : at::zeros_like(u);
  expect("selective_scan", "the gradient of y", gy, u.sizes(), u.device());
  const Tensor du = rows_like(u), dd = rows_like(delta), dz = z.has_value() ? rows_like(*z) : Tensor();
  // without channels nothing is launched, and b and c, whose shapes do not have them, get sums over nothing
  const bool none = u.size(2) == 0;
  const Tensor db = none ? at::zeros(b.sizes(), b.options()) : at::empty(b.sizes(), b.options()),
               dc = none ? at::zeros(c.sizes(), c.options()) : at::empty(c.sizes(), c.options());
  const Tensor da = at::empty(a.sizes(), a.options());
  const Tensor dskip = d.has_value() ? at::empty({u.size(2)}, a.options()) : Tensor(), dbias = bias.has_value() ? at::empty({u.size(2)}, a.options()) : Tensor();
  const Tensor ds = state.has_value() ? at::empty(state->sizes(), state->options()) : Tensor();
  g.dy = view_of(gy, held);
  g.du = view_of(du, held);
  g.ddelta = view_of(dd, held);
  if (dz.defined()) g.dz = view_of(dz, held);
  g.db = shared_view(db, held);
  g.dc = shared_view(dc, held);
  g.dstate_out = floats(dstate, held);
  g.da = static_cast<float*>(da.data_ptr());
  g.dd = dskip.defined() ? static_cast<float*>(dskip.data_ptr()) : nullptr;
  g.ddelta_bias = dbias.defined() ? static_cast<float*>(dbias.data_ptr()) : nullptr;
  g.dstate_in = ds.defined() ? static_cast<float*>(ds.data_ptr()) : nullptr;
  const Tensor scratch = scratch_of(bnb_selective_scan_bwd_scratch_bytes(&k.q), u);
  check("bnb_selective_scan_bwd", bnb_selective_scan_bwd(&k.q, &g, scratch.data_ptr(), (size_t)scratch.numel(), stream_of(u.device())));
  return {du, dd, da, db, dc, dskip, dz, dbias, ds};
}

std::tuple<Tensor, Tensor> scan(const Tensor& u, const Tensor& delta, const Tensor& a, const Tensor& b, const Tensor& c, const OptTensor& d, const OptTensor& z,
                                const OptTensor& bias, const OptTensor& state, const OptTensor& done, const OptTensor& lengths, bool softplus) {
  const variable_list inputs{u, delta, a, b, c, value(d), value(z), value(bias), value(state)};
  Tensor y, out, kept;
  if (!wants_grad(inputs)) {
    std::tie(y, out, kept) = scan_forward(u, delta, a, b, c, d, z, bias, state, done, lengths, softplus, false);
    return {y, out};
  }
  {
    const at::NoGradGuard no_grad;
    std::tie(y, out, kept) = scan_forward(u, delta, a, b, c, d, z, bias, state, done, lengths, softplus, true);
  }
  auto node = node_of(inputs, {value(done), value(lengths), kept}, [softplus](const std::vector<Tensor>& s, const variable_list& g) -> variable_list {
    return scan_backward(s[0], s[1], s[2], s[3], s[4], opt(s[5]), opt(s[6]), opt(s[7]), opt(s[8]), opt(s[9]), opt(s[10]), softplus, s[11], opt(g[0]), opt(g[1]));
  });
  torch::autograd::create_gradient_edge(y, node);
  torch::autograd::create_gradient_edge(out, node);
  return {y, out};
}

Tensor scan_step(const Tensor& u, const Tensor& delta, const Tensor& a, const Tensor& b, const Tensor& c, const OptTensor& d, const Tensor& state, const OptTensor& z,
                 const OptTensor& bias, const OptTensor& reset, bool softplus) {
  const char* fn = "selective_step";
  if (u.dim() != 2) refuse(std::string(fn) + ": u must have shape (R, C), got " + shape_text(u.sizes()));
  const c10::cuda::OptionalCUDAGuard guard(u.is_cuda() ? c10::optional<c10::Device>(u.device()) : c10::nullopt);
  ScanCall k = scan_call(fn, u, delta, a, b, c, d, z, bias, softplus);
  expect_state(fn, state, {u.size(0), u.size(1), a.size(1)}, u.device());
  const OptTensor cleared = reset_bytes(fn, reset, u.size(0), u.device());
  const Tensor y = at::empty(u.sizes(), u.options());
  k.q.y = view_of(y, k.held);
  k.q.state_out = static_cast<float*>(state.data_ptr());
  k.q.state_in = k.q.state_out;
  k.q.reset = data<uint8_t>(cleared);
  check("bnb_selective_step", bnb_selective_step(&k.q, stream_of(u.device())));
  state.unsafeGetTensorImpl()->bump_version();
  return y;
}

// ------------------------------------------------------------------ gated feed-forward block

struct GatedCall {
  BnbGatedBlock c{};
  std::vector<Tensor> held;
};
// x as (rows, width), its rows contiguous elements.
Tensor rows_of(const Tensor& t) {
  const Tensor v = t.reshape({-1, t.size(-1)});
  return v.stride(1) == 1 || v.size(1) <= 1 ? v : v.contiguous();
}
int64_t row_stride(const Tensor& v) { return v.size(0) > 1 ? v.stride(0) : v.size(1); }
GatedCall gated_call(const Tensor& x, const Tensor& gate, const Tensor& up, const Tensor& down, int activation) {
  const char* fn = "gated_mlp";
  expect_cuda(fn, x);
  if (x.dim() < 1) refuse("gated_mlp: x must have shape (.., D)");
  const int64_t D = x.size(-1);
  const c10::Device dev = x.device();
  GatedCall k;
  BnbGatedBlock& c = k.c;
  c.element = element_of(fn, x);
  if (gate.dim() != 2) refuse("gated_mlp: gate_w must have shape (F, " + std::to_string(D) + "), got " + shape_text(gate.sizes()));
  const int64_t F = gate.size(0);
  if (D < 1 || F < 1) throw py::value_error("gated_mlp: width and hidden size must be at least 1");
  expect(fn, "gate_w", gate, {F, D}, dev);
  expect(fn, "up_w", up, {F, D}, dev);
  expect(fn, "down_w", down, {D, F}, dev);
  for (const Tensor* w : {&gate, &up, &down})
    if (w->scalar_type() != gate.scalar_type() || (w->scalar_type() != x.scalar_type() && w->scalar_type() != at::kFloat))
      refuse(std::string("gated_mlp: the weights must all be float32 or all of the input's type ") + c10::toString(x.scalar_type()));
  const Tensor flat = rows_of(x);
  k.held.push_back(flat);
  c.rows = flat.size(0);
  c.width = fits_int(fn, D);
  c.hidden = fits_int(fn, F);
  c.weight_element = element_of(fn, gate);
  c.activation = activation;
  c.x = flat.data_ptr();
  c.x_row = row_stride(flat);
  const void** at[] = {&c.gate_w, &c.up_w, &c.down_w};
  int i = 0;
  for (const Tensor* w : {&gate, &up, &down}) {
    k.held.push_back(contiguous(*w));
    *at[i++] = k.held.back().data_ptr();
  }
  return k;
}

// (y, what the backward reads: empty unless asked for)
std::tuple<Tensor, Tensor> gated_forward(const Tensor& x, const Tensor& gate, const Tensor& up, const Tensor& down, int activation, bool keep) {
  const c10::cuda::OptionalCUDAGuard guard(x.is_cuda() ? c10::optional<c10::Device>(x.device()) : c10::nullopt);
  GatedCall k = gated_call(x, gate, up, down, activation);
  raise_pending_status(x.device());
  const Tensor y = at::empty(x.sizes(), x.options());
  const Tensor kept = at::empty({keep ? (int64_t)bnb_gated_block_kept_bytes(&k.c) : 0}, x.options().dtype(at::kByte));
  k.c.y = y.data_ptr();
  k.c.kept = keep ? kept.data_ptr() : nullptr;
  const Tensor scratch = scratch_of(bnb_gated_block_scratch_bytes(&k.c, 0), x);
  check("bnb_gated_block_fwd", bnb_gated_block_fwd(&k.c, scratch.data_ptr(), (size_t)scratch.numel(), stream_of(x.device())));
  return {y, kept};
}

// Gradients of x, gate_w, up_w and down_w.
std::vector<Tensor> gated_backward(const Tensor& x, const Tensor& gate, const Tensor& up, const Tensor& down, int activation, const Tensor& kept, const Tensor& dy) {
  const c10::cuda::CUDAGuard guard(x.device());
  GatedCall k = gated_call(x, gate, up, down, activation);
  Tensor held = contiguous(kept).to(x.device());
  if (held.scalar_type() != at::kByte || (size_t)held.numel() != bnb_gated_block_kept_bytes(&k.c))
    refuse("gated_mlp: the kept activations came back as another tensor: saved-tensor hooks have to return type and shape as they were");
  if (reinterpret_cast<uintptr_t>(held.data_ptr()) % 16) held = held.clone();
  expect("gated_mlp", "the gradient of y", dy, x.sizes(), x.device());
  const Tensor gy = rows_of(dy.to(x.scalar_type()));
  const Tensor dx = at::empty(x.sizes(), x.options()), dg = at::empty(gate.sizes(), gate.options()), du = at::empty(up.sizes(), up.options()),
               dd = at::empty(down.sizes(), down.options());
  k.c.kept = held.data_ptr();
  const BnbGatedBlockGrads g{gy.data_ptr(), row_stride(gy), dx.data_ptr(), dg.data_ptr(), du.data_ptr(), dd.data_ptr()};
  const Tensor scratch = scratch_of(bnb_gated_block_scratch_bytes(&k.c, 1), x);
  check("bnb_gated_block_bwd", bnb_gated_block_bwd(&k.c, &g, scratch.data_ptr(), (size_t)scratch.numel(), stream_of(x.device())));
  return {dx, dg, du, dd};
}

Tensor gated(const Tensor& x, const Tensor& gate, const Tensor& up, const Tensor& down, int activation) {
  const variable_list inputs{x, gate, up, down};
  if (!wants_grad(inputs)) return std::get<0>(gated_forward(x, gate, up, down, activation, false));
  Tensor y, kept;
  {
    const at::NoGradGuard no_grad;
    std::tie(y, kept) = gated_forward(x, gate, up, down, activation, true);
  }
  auto node = node_of(inputs, {kept}, [activation](const std::vector<Tensor>& s, const variable_list& g) -> variable_list {
    if (!g[0].defined()) return variable_list(4);
    return gated_backward(s[0], s[1], s[2], s[3], activation, s[4], g[0]);
  });
  torch::autograd::create_gradient_edge(y, node);
  return y;
}

}  // namespace

void bind_operators(py::module& m) {
  m.def("causal_conv_forward", &conv_forward);
  m.def("causal_conv_backward", &conv_backward);
  m.def("causal_conv", torch::wrap_pybind_function(conv));
  m.def("causal_conv_step", &conv_step);
  m.def("selective_scan_forward", &scan_forward);
  m.def("selective_scan_backward", &scan_backward);
  m.def("selective_scan", torch::wrap_pybind_function(scan));
  m.def("selective_step", &scan_step);
  m.def("gated_mlp_forward", &gated_forward);
  m.def("gated_mlp_backward", &gated_backward);
  m.def("gated_mlp", torch::wrap_pybind_function(gated));
}

}  // namespace host
}  // namespace bnb
