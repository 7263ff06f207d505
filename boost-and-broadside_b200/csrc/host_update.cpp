// The host side of the operators behind the trunk in an update (yemong/linear.py, yemong/policy_loss.py, yemong/optimizer.py): checks, outputs and scratch from torch's
// allocator, the launch, the autograd nodes of eager calls.
#include "host_nodes.h"

#include <torch/csrc/autograd/python_variable.h>

#include <tuple>

namespace bnb {
namespace host {
namespace {

// ------------------------------------------------------------------ linear layer

struct LinearCall {
  BnbLinear c{};
  std::vector<Tensor> held;
};
std::vector<int64_t> out_sizes(const Tensor& x, const Tensor& weight) {
  std::vector<int64_t> s = x.sizes().vec();
  s.back() = weight.size(0);
  return s;
}
LinearCall linear_call(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& residual, int activation) {
  const char* fn = "linear";
  expect_cuda(fn, x);
  if (x.dim() < 1) refuse("linear: x must have shape (.., width)");
  const int64_t K = x.size(-1);
  const c10::Device dev = x.device();
  LinearCall k;
  BnbLinear& c = k.c;
  c.element = element_of(fn, x);
  if (weight.dim() != 2) refuse("linear: weight must have shape (out, " + std::to_string(K) + "), got " + shape_text(weight.sizes()));
  const int64_t N = weight.size(0);
  if (K < 1 || N < 1) throw py::value_error("linear: width and outputs must be at least 1");
  expect(fn, "weight", weight, {N, K}, dev);
  if (weight.scalar_type() != x.scalar_type() && weight.scalar_type() != at::kFloat)
    refuse(std::string("linear: weight must be float32 or of the input's type ") + c10::toString(x.scalar_type()));
  c.weight_element = element_of(fn, weight);
  c.bias_element = c.element;
  if (bias.has_value()) {
    expect(fn, "bias", *bias, {N}, dev);
    if (bias->scalar_type() != x.scalar_type() && bias->scalar_type() != at::kFloat)
      refuse(std::string("linear: bias must be float32 or of the input's type ") + c10::toString(x.scalar_type()));
    c.bias_element = element_of(fn, *bias);
    k.held.push_back(contiguous(*bias));
    c.bias = k.held.back().data_ptr();
  }
  const Tensor flat = rows_of(x);
  k.held.push_back(flat);
  c.rows = flat.size(0);
  c.width = fits_int(fn, K);
  c.out = fits_int(fn, N);
  c.activation = activation;
  c.x = flat.data_ptr();
  c.x_row = row_stride(flat);
  k.held.push_back(contiguous(weight));
  c.weight = k.held.back().data_ptr();
  if (residual.has_value()) {
    expect(fn, "residual", *residual, out_sizes(x, weight), dev);
    expect_type(fn, "residual", *residual, x.scalar_type());
    const Tensor r = rows_of(*residual);
    k.held.push_back(r);
    c.residual = r.data_ptr();
    c.residual_row = row_stride(r);
  }
  return k;
}

// (y, what the backward reads: empty unless asked for)
std::tuple<Tensor, Tensor> linear_forward(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& residual, int activation, bool keep) {
  const c10::cuda::OptionalCUDAGuard guard(x.is_cuda() ? c10::optional<c10::Device>(x.device()) : c10::nullopt);
  LinearCall k = linear_call(x, weight, bias, residual, activation);
  raise_pending_status(x.device());
  const Tensor y = at::empty(out_sizes(x, weight), x.options());
  const Tensor kept = at::empty({keep ? (int64_t)bnb_linear_kept_bytes(&k.c) : 0}, x.options().dtype(at::kByte));
  k.c.y = y.data_ptr();
  k.c.kept = keep && kept.numel() ? kept.data_ptr() : nullptr;
  const Tensor scratch = scratch_of(bnb_linear_scratch_bytes(&k.c, 0), x);
  check("bnb_linear_fwd", bnb_linear_fwd(&k.c, scratch.data_ptr(), (size_t)scratch.numel(), stream_of(x.device())));
  return {y, kept};
}

// Gradients of x, weight and bias, those that are wanted.
std::vector<Tensor> linear_backward(const Tensor& x, const Tensor& weight, const OptTensor& bias, int activation, const Tensor& kept, const Tensor& dy,
                                    bool want_x, bool want_weight, bool want_bias) {
  if (!want_x && !want_weight && !(want_bias && bias.has_value())) return std::vector<Tensor>(3);
  const c10::cuda::CUDAGuard guard(x.device());
  LinearCall k = linear_call(x, weight, bias, c10::nullopt, activation);
  Tensor held = contiguous(kept).to(x.device());
  if (held.scalar_type() != at::kByte || (size_t)held.numel() != bnb_linear_kept_bytes(&k.c))
    refuse("linear: the kept activations came back as another tensor: saved-tensor hooks have to return type and shape as they were");
  if (reinterpret_cast<uintptr_t>(held.data_ptr()) % 16) held = held.clone();
  expect("linear", "the gradient of y", dy, out_sizes(x, weight), x.device());
  const Tensor gy = rows_of(dy.to(x.scalar_type()));
  const Tensor dx = want_x ? at::empty(x.sizes(), x.options()) : Tensor(), dw = want_weight ? at::empty(weight.sizes(), weight.options()) : Tensor(),
               db = want_bias && bias.has_value() ? at::empty(bias->sizes(), bias->options()) : Tensor();
  auto at_ = [](const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
  k.c.kept = held.numel() ? held.data_ptr() : nullptr;
  const BnbLinearGrads g{gy.data_ptr(), row_stride(gy), at_(dx), at_(dw), at_(db)};
  const Tensor scratch = scratch_of(bnb_linear_scratch_bytes(&k.c, 1), x);
  check("bnb_linear_bwd", bnb_linear_bwd(&k.c, &g, scratch.data_ptr(), (size_t)scratch.numel(), stream_of(x.device())));
  return {dx, dw, db};
}

Tensor linear(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& residual, int activation) {
  const variable_list inputs{x, weight, value(bias), value(residual)};
  if (!wants_grad(inputs)) return std::get<0>(linear_forward(x, weight, bias, residual, activation, false));
  Tensor y, kept;
  {
    const at::NoGradGuard no_grad;
    std::tie(y, kept) = linear_forward(x, weight, bias, residual, activation, true);
  }
  // the residual's values are not needed again: an undefined tensor in its place
  auto node = node_of({x, weight, value(bias)}, {kept}, {});
  node->set_next_edges(torch::autograd::collect_next_edges(inputs));
  const bool has_residual = residual.has_value();
  OpNode* const self = node.get();
  node->backward = [activation, has_residual, self](const std::vector<Tensor>& s, const variable_list& g) -> variable_list {
    if (!g[0].defined()) return variable_list(4);
    variable_list out = linear_backward(s[0], s[1], opt(s[2]), activation, s[3], g[0], self->task_should_compute_output(0), self->task_should_compute_output(1),
                                        s[2].defined() && self->task_should_compute_output(2));
    out.push_back(has_residual ? g[0].to(s[0].scalar_type()) : Tensor());
    return out;
  };
  torch::autograd::create_gradient_edge(y, node);
  return y;
}

// ------------------------------------------------------------------ policy loss

struct PolicyCall {
  BnbPolicyLoss c{};
  std::vector<Tensor> held;
};
// A value a row, as contiguous float32.
const float* row_values(const char* name, const Tensor& t, at::IntArrayRef lead, const c10::Device& dev, std::vector<Tensor>& held) {
  expect("policy_loss", name, t, lead, dev);
  if (!t.is_floating_point()) refuse(std::string("policy_loss: ") + name + " must be floating point, got " + c10::toString(t.scalar_type()));
  held.push_back(contiguous(t.to(at::kFloat)));
  return static_cast<const float*>(held.back().data_ptr());
}
// sizes: empty for one slice of all logits, whose actions have no dimension of their own.
PolicyCall policy_call(const Tensor& logits, const Tensor& actions, const Tensor& old_logprob, const Tensor& advantages, const OptTensor& ref_logprob,
                       const OptTensor& weights, const std::vector<int64_t>& sizes, double clip_low, double clip_high, double kl_coef, double entropy_coef) {
  const char* fn = "policy_loss";
  expect_cuda(fn, logits);
  if (logits.dim() < 1 || logits.size(-1) < 1) refuse("policy_loss: logits must have shape (.., actions), got " + shape_text(logits.sizes()));
  const c10::Device dev = logits.device();
  PolicyCall k;
  BnbPolicyLoss& c = k.c;
  c.element = element_of(fn, logits);
  const at::IntArrayRef lead = logits.sizes().slice(0, logits.dim() - 1);
  std::vector<int64_t> per_action = lead.vec();
  const std::vector<int64_t> all{logits.size(-1)};
  const std::vector<int64_t>& slices = sizes.empty() ? all : sizes;
  if (!sizes.empty()) per_action.push_back((int64_t)sizes.size());
  if (slices.size() > BNB_MAX_SLICES) throw py::value_error("policy_loss: at most " + std::to_string(BNB_MAX_SLICES) + " slices are built, got " + std::to_string(slices.size()));
  int64_t width = 0;
  for (int64_t n : slices) {
    if (n < 1) throw py::value_error("policy_loss: every slice needs an action");
    width += n;
  }
  if (width != logits.size(-1))
    throw py::value_error("policy_loss: the slices have " + std::to_string(width) + " actions, the logits " + std::to_string(logits.size(-1)));
  c.n_slices = (int)slices.size();
  for (size_t i = 0; i < slices.size(); ++i) c.sizes[i] = fits_int(fn, slices[i]);
  expect(fn, "actions", actions, per_action, dev);
  if (actions.scalar_type() != at::kLong && actions.scalar_type() != at::kInt) refuse("policy_loss: actions must be int64 or int32");
  k.held.push_back(contiguous(actions.to(at::kLong)));
  c.actions = static_cast<const int64_t*>(k.held.back().data_ptr());
  const Tensor flat = rows_of(logits);
  k.held.push_back(flat);
  c.rows = flat.size(0);
  c.logits = flat.data_ptr();
  c.logits_row = row_stride(flat);
  c.old_logprob = row_values("old_logprob", old_logprob, lead, dev, k.held);
  c.advantages = row_values("advantages", advantages, lead, dev, k.held);
  if (ref_logprob.has_value()) c.ref_logprob = row_values("ref_logprob", *ref_logprob, lead, dev, k.held);
  if (weights.has_value()) {
    if (weights->scalar_type() == at::kBool) {
      expect(fn, "weights", *weights, lead, dev);
      k.held.push_back(contiguous(*weights));
      c.mask = static_cast<const uint8_t*>(k.held.back().data_ptr());
    } else {
      c.weights = row_values("weights", *weights, lead, dev, k.held);
    }
  }
  c.clip_low = (float)clip_low;
  c.clip_high = (float)clip_high;
  c.kl_coef = (float)kl_coef;
  c.entropy_coef = (float)entropy_coef;
  return k;
}

// (loss, log-probability of each row's actions, means, what the backward reads)
std::tuple<Tensor, Tensor, Tensor, Tensor> policy_forward(const Tensor& logits, const Tensor& actions, const Tensor& old_logprob, const Tensor& advantages,
                                                          const OptTensor& ref_logprob, const OptTensor& weights, const std::vector<int64_t>& sizes,
                                                          double clip_low, double clip_high, double kl_coef, double entropy_coef) {
  const c10::cuda::OptionalCUDAGuard guard(logits.is_cuda() ? c10::optional<c10::Device>(logits.device()) : c10::nullopt);
  PolicyCall k = policy_call(logits, actions, old_logprob, advantages, ref_logprob, weights, sizes, clip_low, clip_high, kl_coef, entropy_coef);
  const auto floats_of = logits.options().dtype(at::kFloat);
  const Tensor loss = at::empty({}, floats_of), stats = at::empty({4}, floats_of), logprob = at::empty(old_logprob.sizes(), floats_of);
  const Tensor kept = at::empty({(int64_t)(bnb_policy_loss_kept_bytes(&k.c) / 4)}, floats_of);
  k.c.loss = static_cast<float*>(loss.data_ptr());
  k.c.stats = static_cast<float*>(stats.data_ptr());
  k.c.logprob = static_cast<float*>(logprob.data_ptr());
  k.c.kept = static_cast<float*>(kept.data_ptr());
  const Tensor scratch = scratch_of(bnb_policy_loss_scratch_bytes(&k.c), logits);
  check("bnb_policy_loss_fwd", bnb_policy_loss_fwd(&k.c, scratch.data_ptr(), (size_t)scratch.numel(), stream_of(logits.device())));
  return {loss, logprob, stats, kept};
}

Tensor policy_backward(const Tensor& logits, const Tensor& actions, const Tensor& old_logprob, const Tensor& advantages, const OptTensor& ref_logprob,
                       const OptTensor& weights, const std::vector<int64_t>& sizes, double clip_low, double clip_high, double kl_coef, double entropy_coef,
                       const Tensor& kept, const Tensor& dloss) {
  const c10::cuda::CUDAGuard guard(logits.device());
  PolicyCall k = policy_call(logits, actions, old_logprob, advantages, ref_logprob, weights, sizes, clip_low, clip_high, kl_coef, entropy_coef);
  const Tensor rows = contiguous(kept).to(logits.device());
  if (rows.scalar_type() != at::kFloat || (size_t)rows.numel() * 4 != bnb_policy_loss_kept_bytes(&k.c))
    refuse("policy_loss: what the forward kept came back as another tensor: saved-tensor hooks have to return type and shape as they were");
  expect("policy_loss", "the gradient of the loss", dloss, {}, logits.device());
  const Tensor slope = dloss.to(at::kFloat);
  const Tensor out = at::empty(logits.sizes(), logits.options());
  k.c.kept = static_cast<float*>(rows.data_ptr());
  check("bnb_policy_loss_bwd", bnb_policy_loss_bwd(&k.c, static_cast<const float*>(slope.data_ptr()), out.data_ptr(), stream_of(logits.device())));
  return out;
}

std::tuple<Tensor, Tensor, Tensor> policy_loss(const Tensor& logits, const Tensor& actions, const Tensor& old_logprob, const Tensor& advantages,
                                               const OptTensor& ref_logprob, const OptTensor& weights, const std::vector<int64_t>& sizes, double clip_low,
                                               double clip_high, double kl_coef, double entropy_coef) {
  const variable_list inputs{logits};
  Tensor loss, logprob, stats, kept;
  {
    const at::NoGradGuard no_grad;
    std::tie(loss, logprob, stats, kept) =
        policy_forward(logits, actions, old_logprob, advantages, ref_logprob, weights, sizes, clip_low, clip_high, kl_coef, entropy_coef);
  }
  if (!wants_grad(inputs)) return {loss, logprob, stats};
  auto node = node_of(inputs, {actions, old_logprob, advantages, value(ref_logprob), value(weights), kept},
                      [=](const std::vector<Tensor>& s, const variable_list& g) -> variable_list {
                        if (!g[0].defined()) return variable_list(1);
                        return {policy_backward(s[0], s[1], s[2], s[3], opt(s[4]), opt(s[5]), sizes, clip_low, clip_high, kl_coef, entropy_coef, s[6], g[0])};
                      });
  torch::autograd::create_gradient_edge(loss, node);
  return {loss, logprob, stats};
}

// ------------------------------------------------------------------ AdamW

constexpr int64_t STATE_BLOCK = 256;   // elements that share a scale of 8-bit states

bool laid_out_as(const Tensor& t, const Tensor& p) { return t.sizes() == p.sizes() && (t.strides() == p.strides() || (t.is_contiguous() && p.is_contiguous())); }
Tensor state_of(const py::dict& state, const char* name) {
  PyObject* v = PyDict_GetItemString(state.ptr(), name);
  if (!v || !THPVariable_Check(v)) refuse(std::string("AdamW: a parameter's state has no tensor '") + name + "'");
  return THPVariable_Unpack(v);
}
void expect_kept(const char* name, const Tensor& t, const Tensor& like, at::ScalarType type, const c10::Device& dev) {
  if (t.scalar_type() != type || t.device() != dev || !laid_out_as(t, like))
    refuse(std::string("AdamW: the state '") + name + "' must be " + c10::toString(type) + " of shape " + shape_text(like.sizes()) + " on " + dev.str() +
           ", laid out as its parameter; got " + c10::toString(t.scalar_type()) + " of shape " + shape_text(t.sizes()) + " on " + t.device().str());
}
void expect_changeable(const char* name, const Tensor& t) {
  if (t.is_inference() && !c10::InferenceMode::is_enabled())
    refuse(std::string("AdamW: ") + name + " was made in inference mode, outside of which it must not be changed");
}

// One step of the parameters of all groups that have a gradient.  groups: (parameters, states: dicts of tensors, positions, lr, beta1, beta2, eps, weight decay)
// each.  Everything is checked before the first launch.  Returns the gradients' norm where they are clipped.
using Group = std::tuple<py::list, py::list, std::vector<int64_t>, py::object, double, double, double, double>;
OptTensor adamw_step(const std::vector<Group>& groups, const py::object& max_norm, int state_bits, uint32_t seed, const Tensor& control) {
  const bool eight = state_bits == 8;
  std::vector<Tensor> held, changed;
  std::vector<std::vector<BnbAdamTensor>> lists;
  std::vector<BnbAdamW> calls;
  c10::optional<c10::Device> dev;
  for (const Group& group : groups) {
    const auto& [params, states, positions, lr, beta1, beta2, eps, decay] = group;
    std::vector<BnbAdamTensor> list;
    for (size_t i = 0; i < params.size(); ++i) {
      const Tensor p = THPVariable_Unpack(params[i].ptr());
      Tensor g = p.grad();
      if (!g.defined()) continue;
      if (!p.is_cuda()) refuse("AdamW: a parameter is on " + p.device().str() + "; the kernels run on CUDA only (sm_100a) and have no CPU path");
      if (!dev) dev = p.device();
      if (p.device() != *dev) refuse("AdamW: parameters on " + p.device().str() + " and " + dev->str() + "; one optimizer serves one device");
      if (g.layout() != at::kStrided) refuse("AdamW: sparse gradients are not taken");
      if (g.scalar_type() != p.scalar_type() || g.sizes() != p.sizes() || g.device() != *dev) refuse("AdamW: a gradient has another type, shape or device than its parameter");
      if (!p.is_non_overlapping_and_dense()) throw py::value_error("AdamW: a parameter's elements must lie densely in memory, each in a place of its own");
      const c10::cuda::CUDAGuard guard(*dev);
      BnbAdamTensor t{};
      t.element = element_of("AdamW", p);
      t.n = p.numel();
      t.position = positions[i];
      const py::dict state = py::reinterpret_borrow<py::dict>(states[i]);
      const Tensor step = state_of(state, "step"), m = state_of(state, "exp_avg"), v = state_of(state, eight ? "exp_avg_sq_root" : "exp_avg_sq");
      if (step.scalar_type() != at::kFloat || step.numel() != 1 || step.device() != *dev) refuse("AdamW: the state 'step' must be one float32 number on " + dev->str());
      const at::ScalarType type = eight ? at::kFloat8_e4m3fn : at::kFloat;
      expect_kept("exp_avg", m, p, type, *dev);
      expect_kept(eight ? "exp_avg_sq_root" : "exp_avg_sq", v, p, type, *dev);
      if (eight) {
        const int64_t blocks = (t.n + STATE_BLOCK - 1) / STATE_BLOCK;
        for (const auto& [name, to] : {std::pair<const char*, float**>{"exp_avg_scale", &t.m_scale}, {"exp_avg_sq_root_scale", &t.v_scale}}) {
          const Tensor s = state_of(state, name);
          if (s.scalar_type() != at::kFloat || s.dim() != 1 || s.size(0) != blocks || !s.is_contiguous() || s.device() != *dev)
            refuse(std::string("AdamW: the state '") + name + "' must be float32 of shape " + shape_text({blocks}) + ", contiguous, on " + dev->str());
          *to = static_cast<float*>(s.data_ptr());
          changed.push_back(s);
        }
      }
      if (!laid_out_as(g, p)) {
        g = at::empty_like(p).copy_(g);
        held.push_back(g);
      }
      t.p = p.data_ptr();
      t.g = g.data_ptr();
      t.m = m.data_ptr();
      t.v = v.data_ptr();
      t.step = static_cast<float*>(step.data_ptr());
      list.push_back(t);
      changed.insert(changed.end(), {p, m, v, step});
    }
    BnbAdamW c{};
    c.state_bits = state_bits;
    c.seed = seed;
    if (THPVariable_Check(lr.ptr())) {
      const Tensor rate = THPVariable_Unpack(lr.ptr());
      if (rate.numel() != 1) refuse("AdamW: lr must be a number or a tensor of one");
      if (rate.is_cuda()) {
        if (dev && rate.device() != *dev) refuse("AdamW: lr is on " + rate.device().str() + ", the parameters on " + dev->str());
        held.push_back(rate.to(at::kFloat));
        c.lr_device = static_cast<const float*>(held.back().data_ptr());
      } else {
        c.lr = rate.item<float>();
      }
    } else {
      c.lr = (float)lr.cast<double>();
    }
    c.beta1 = beta1;
    c.beta2 = beta2;
    c.eps = (float)eps;
    c.weight_decay = (float)decay;
    c.control = static_cast<int32_t*>(control.data_ptr());
    calls.push_back(c);
    lists.push_back(std::move(list));
  }
  if (!dev) return c10::nullopt;
  expect("AdamW", "the control word", control, {1}, *dev);
  for (const Tensor& t : changed) expect_changeable("a parameter or its state", t);
  const c10::cuda::CUDAGuard guard(*dev);
  void* stream = stream_of(*dev);
  OptTensor norm;
  Tensor parts;
  if (!max_norm.is_none()) {
    const auto options = at::TensorOptions().device(*dev);
    parts = at::empty({BNB_GRAD_NORM_PARTS}, options.dtype(at::kDouble));
    norm = at::empty({}, options.dtype(at::kFloat));
    std::vector<BnbAdamTensor> all;
    for (const auto& list : lists) all.insert(all.end(), list.begin(), list.end());
    check("bnb_grad_norm", bnb_grad_norm(all.data(), (int)all.size(), static_cast<double*>(parts.data_ptr()), stream));
  }
  for (size_t i = 0; i < lists.size(); ++i) {
    if (norm.has_value()) {
      calls[i].norm_parts = static_cast<const double*>(parts.data_ptr());
      calls[i].n_norm_parts = BNB_GRAD_NORM_PARTS;
      calls[i].max_norm = (float)max_norm.cast<double>();
      calls[i].norm = static_cast<float*>(norm->data_ptr());
    }
    check("bnb_adamw_step", bnb_adamw_step(lists[i].data(), (int)lists[i].size(), &calls[i], stream));
  }
  for (const Tensor& t : changed)
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  return norm;
}

}  // namespace

void bind_update(py::module& m) {
  m.def("linear_forward", &linear_forward);
  m.def("linear_backward", &linear_backward);
  m.def("linear", torch::wrap_pybind_function(linear));
  m.def("adamw_step", &adamw_step);
  m.def("policy_loss_forward", &policy_forward);
  m.def("policy_loss_backward", &policy_backward);
  m.def("policy_loss", torch::wrap_pybind_function(policy_loss));
}

}  // namespace host
}  // namespace bnb
