// The host side of the operators behind the trunk in an update (yemong/linear.py, yemong/policy_loss.py, yemong/optimizer.py): checks, outputs and scratch from torch's
// allocator, the launch, the autograd nodes of eager calls.
#include "host_nodes.h"

#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
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

struct PolicyResults { Tensor loss, logprob, stats, kept, dlogits; };
// gradients: the logits' for dloss = 1 are written too, where the call takes them.
PolicyResults policy_results(const Tensor& logits, const Tensor& actions, const Tensor& old_logprob, const Tensor& advantages,
                             const OptTensor& ref_logprob, const OptTensor& weights, const std::vector<int64_t>& sizes, double clip_low, double clip_high,
                             double kl_coef, double entropy_coef, bool gradients) {
  const c10::cuda::OptionalCUDAGuard guard(logits.is_cuda() ? c10::optional<c10::Device>(logits.device()) : c10::nullopt);
  PolicyCall k = policy_call(logits, actions, old_logprob, advantages, ref_logprob, weights, sizes, clip_low, clip_high, kl_coef, entropy_coef);
  const auto floats_of = logits.options().dtype(at::kFloat);
  const Tensor loss = at::empty({}, floats_of), stats = at::empty({4}, floats_of), logprob = at::empty(old_logprob.sizes(), floats_of);
  const Tensor kept = at::empty({(int64_t)(bnb_policy_loss_kept_bytes(&k.c) / 4)}, floats_of);
  k.c.loss = static_cast<float*>(loss.data_ptr());
  k.c.stats = static_cast<float*>(stats.data_ptr());
  k.c.logprob = static_cast<float*>(logprob.data_ptr());
  k.c.kept = static_cast<float*>(kept.data_ptr());
  const Tensor dlogits = gradients && bnb_policy_loss_takes_gradients(&k.c) ? at::empty(logits.sizes(), logits.options()) : Tensor();
  k.c.dlogits = dlogits.defined() && dlogits.numel() ? dlogits.data_ptr() : nullptr;
  const Tensor scratch = scratch_of(bnb_policy_loss_scratch_bytes(&k.c), logits);
  check("bnb_policy_loss_fwd", bnb_policy_loss_fwd(&k.c, scratch.data_ptr(), (size_t)scratch.numel(), stream_of(logits.device())));
  return {loss, logprob, stats, kept, dlogits};
}
// (loss, log-probability of each row's actions, means, what the backward reads)
std::tuple<Tensor, Tensor, Tensor, Tensor> policy_forward(const Tensor& logits, const Tensor& actions, const Tensor& old_logprob, const Tensor& advantages,
                                                          const OptTensor& ref_logprob, const OptTensor& weights, const std::vector<int64_t>& sizes,
                                                          double clip_low, double clip_high, double kl_coef, double entropy_coef) {
  const PolicyResults r = policy_results(logits, actions, old_logprob, advantages, ref_logprob, weights, sizes, clip_low, clip_high, kl_coef, entropy_coef, false);
  return {r.loss, r.logprob, r.stats, r.kept};
}

Tensor policy_backward(const Tensor& logits, const Tensor& actions, const Tensor& old_logprob, const Tensor& advantages, const OptTensor& ref_logprob,
                       const OptTensor& weights, const std::vector<int64_t>& sizes, double clip_low, double clip_high, double kl_coef, double entropy_coef,
                       const Tensor& kept, const Tensor& dloss, const Tensor& unit) {
  const c10::cuda::CUDAGuard guard(logits.device());
  PolicyCall k = policy_call(logits, actions, old_logprob, advantages, ref_logprob, weights, sizes, clip_low, clip_high, kl_coef, entropy_coef);
  const Tensor rows = contiguous(kept).to(logits.device());
  if (rows.scalar_type() != at::kFloat || (size_t)rows.numel() * 4 != bnb_policy_loss_kept_bytes(&k.c))
    refuse("policy_loss: what the forward kept came back as another tensor: saved-tensor hooks have to return type and shape as they were");
  expect("policy_loss", "the gradient of the loss", dloss, {}, logits.device());
  const Tensor slope = dloss.to(at::kFloat);
  // the gradient that the forward wrote, if it is as it was
  const bool holds = unit.defined() && unit.sizes() == logits.sizes() && unit.scalar_type() == logits.scalar_type() && unit.device() == logits.device() &&
                     unit.is_contiguous() && reinterpret_cast<uintptr_t>(unit.data_ptr()) % 16 == 0;
  const Tensor out = holds ? unit : at::empty(logits.sizes(), logits.options());
  k.c.kept = static_cast<float*>(rows.data_ptr());
  check("bnb_policy_loss_bwd", bnb_policy_loss_bwd(&k.c, static_cast<const float*>(slope.data_ptr()), out.data_ptr(), holds ? 1 : 0, stream_of(logits.device())));
  return out;
}
Tensor policy_backward_alone(const Tensor& logits, const Tensor& actions, const Tensor& old_logprob, const Tensor& advantages, const OptTensor& ref_logprob,
                             const OptTensor& weights, const std::vector<int64_t>& sizes, double clip_low, double clip_high, double kl_coef, double entropy_coef,
                             const Tensor& kept, const Tensor& dloss) {
  return policy_backward(logits, actions, old_logprob, advantages, ref_logprob, weights, sizes, clip_low, clip_high, kl_coef, entropy_coef, kept, dloss, Tensor());
}
// The capture that a device's current stream is in, or 0.
unsigned long long capture_of(const c10::Device& dev) {
  cudaStreamCaptureStatus status;
  unsigned long long id = 0;
  if (cudaStreamGetCaptureInfo(at::cuda::getCurrentCUDAStream(dev.index()).stream(), &status, &id) != cudaSuccess) {
    (void)cudaGetLastError();
    return 0;
  }
  return status == cudaStreamCaptureStatusActive ? id : 0;
}

std::tuple<Tensor, Tensor, Tensor> policy_loss(const Tensor& logits, const Tensor& actions, const Tensor& old_logprob, const Tensor& advantages,
                                               const OptTensor& ref_logprob, const OptTensor& weights, const std::vector<int64_t>& sizes, double clip_low,
                                               double clip_high, double kl_coef, double entropy_coef, bool grad_in_forward) {
  const variable_list inputs{logits};
  const bool differentiable = wants_grad(inputs);
  PolicyResults r;
  {
    const at::NoGradGuard no_grad;
    r = policy_results(logits, actions, old_logprob, advantages, ref_logprob, weights, sizes, clip_low, clip_high, kl_coef, entropy_coef,
                       differentiable && grad_in_forward);
  }
  if (!differentiable) return {r.loss, r.logprob, r.stats};
  auto node = node_of(inputs, {actions, old_logprob, advantages, value(ref_logprob), value(weights), r.kept, r.dlogits}, {});
  OpNode* const self = node.get();
  // The gradient that the forward wrote goes out once: a second backward of the same graph, or one whose forward is not part of its
  // capture (a replay has to repeat it), computes it.
  const unsigned long long capture = capture_of(logits.device());
  node->backward = [=](const std::vector<Tensor>& s, const variable_list& g) -> variable_list {
    if (!g[0].defined()) return variable_list(1);
    self->saved[7] = SavedVariable();
    const Tensor unit = s[7].defined() && capture_of(s[0].device()) == capture ? s[7] : Tensor();
    return {policy_backward(s[0], s[1], s[2], s[3], opt(s[4]), opt(s[5]), sizes, clip_low, clip_high, kl_coef, entropy_coef, s[6], g[0], unit)};
  };
  torch::autograd::create_gradient_edge(r.loss, node);
  return {r.loss, r.logprob, r.stats};
}

// ------------------------------------------------------------------ AdamW

constexpr int64_t STATE_BLOCK = 256;   // elements that share a scale of 8-bit states

bool laid_out_as(const Tensor& t, const Tensor& p) { return t.sizes() == p.sizes() && (t.strides() == p.strides() || (t.is_contiguous() && p.is_contiguous())); }
void expect_kept(const char* name, const Tensor& t, const Tensor& like, at::ScalarType type, const c10::Device& dev) {
  if (t.scalar_type() != type || t.device() != dev || !laid_out_as(t, like))
    refuse(std::string("AdamW: the state '") + name + "' must be " + c10::toString(type) + " of shape " + shape_text(like.sizes()) + " on " + dev.str() +
           ", laid out as its parameter; got " + c10::toString(t.scalar_type()) + " of shape " + shape_text(t.sizes()) + " on " + t.device().str());
}
void expect_changeable(const Tensor& t) {
  if (t.is_inference() && !c10::InferenceMode::is_enabled())
    refuse("AdamW: a parameter or its state was made in inference mode, outside of which it must not be changed");
}

// The parameters and states of an optimizer as tensors, looked up once: a hundred of them cost more in Python than their update on the GPU.  A step
// compares the optimizer's lists and dicts with those that the plan was made of, object by object, so what was replaced in them is seen; what
// may change in place (data, types, gradients) is read anew.
class AdamWPlan {
 public:
  AdamWPlan(const py::list& groups, const py::dict& state, int state_bits) : eight_(state_bits == 8) {
    names_ = eight_ ? std::vector<const char*>{"step", "exp_avg", "exp_avg_sq_root", "exp_avg_scale", "exp_avg_sq_root_scale"}
                    : std::vector<const char*>{"step", "exp_avg", "exp_avg_sq"};
    for (const char* name : names_) keys_.push_back(py::reinterpret_steal<py::object>(PyUnicode_InternFromString(name)));
    int64_t at = 0;
    for (const py::handle& group : groups) {
      std::vector<Entry> entries;
      for (const py::handle& param : py::list(group["params"])) {
        Entry e;
        e.object = py::reinterpret_borrow<py::object>(param);
        e.p = THPVariable_Unpack(param.ptr());
        e.position = at;
        at += (e.p.numel() + STATE_BLOCK - 1) / STATE_BLOCK * STATE_BLOCK;
        PyObject* of = PyDict_GetItemWithError(state.ptr(), param.ptr());
        if (!of && PyErr_Occurred()) throw py::error_already_set();
        if (of && PyDict_Check(of) && PyDict_Size(of)) {
          e.state = py::reinterpret_borrow<py::object>(of);
          for (size_t i = 0; i < names_.size(); ++i) {
            PyObject* v = PyDict_GetItemWithError(of, keys_[i].ptr());
            if (!v || !THPVariable_Check(v)) refuse(std::string("AdamW: a parameter's state has no tensor '") + names_[i] + "'");
            e.objects.push_back(py::reinterpret_borrow<py::object>(v));
            e.kept.push_back(THPVariable_Unpack(v));
          }
        }
        entries.push_back(std::move(e));
      }
      groups_.push_back(std::move(entries));
    }
    // elements of two parameters at one place would be updated at the same time
    std::vector<std::pair<uintptr_t, uintptr_t>> places;
    for (const auto& entries : groups_)
      for (const Entry& e : entries)
        if (e.p.numel() && e.p.is_non_overlapping_and_dense()) {
          const auto at = reinterpret_cast<uintptr_t>(e.p.data_ptr());
          places.emplace_back(at, at + e.p.numel() * e.p.element_size());
        }
    std::sort(places.begin(), places.end());
    for (size_t i = 1; i < places.size(); ++i)
      if (places[i].first < places[i - 1].second) throw py::value_error("AdamW: two parameters share memory");
    PyObject *key, *value;
    for (Py_ssize_t i = 0; PyDict_Next(state.ptr(), &i, &key, &value);) states_.emplace_back(py::reinterpret_borrow<py::object>(key), py::reinterpret_borrow<py::object>(value));
  }

  // One step of the parameters that have a gradient.  False where the plan is of other lists, dicts or states than these; else the gradients' norm where
  // they are clipped, or None.  Everything is checked before the first launch.
  py::object step(const py::list& groups, const py::dict& state, const py::object& max_norm, uint32_t seed, const Tensor& control) {
    if (!is_of(groups, state)) return py::bool_(false);
    std::vector<Tensor> held;
    std::vector<const Tensor*> changed;
    std::vector<std::vector<BnbAdamTensor>> lists(groups_.size());
    std::vector<BnbAdamW> calls(groups_.size());
    const c10::Device dev = control.device();
    const c10::cuda::OptionalCUDAGuard guard(control.is_cuda() ? c10::optional<c10::Device>(dev) : c10::nullopt);
    size_t total = 0;
    for (size_t i = 0; i < groups_.size(); ++i) {
      const py::dict group = groups[i];
      for (const Entry& e : groups_[i])
        if (const Tensor& g = e.p.grad(); g.defined()) lists[i].push_back(tensor_of(e, g, dev, held, changed));
      calls[i] = call_of(group, seed, control, held);
      total += lists[i].size();
    }
    if (!total) return py::none();
    expect("AdamW", "the control word", control, {1}, dev);
    for (const Tensor* t : changed) expect_changeable(*t);
    void* stream = stream_of(dev);
    py::object out = py::none();
    Tensor parts, norm;
    if (!max_norm.is_none()) {
      parts = at::empty({BNB_GRAD_NORM_PARTS}, control.options().dtype(at::kDouble));
      norm = at::empty({}, control.options().dtype(at::kFloat));
      std::vector<BnbAdamTensor> all;
      if (lists.size() > 1)
        for (const auto& list : lists) all.insert(all.end(), list.begin(), list.end());
      const std::vector<BnbAdamTensor>& of = lists.size() > 1 ? all : lists[0];
      check("bnb_grad_norm", bnb_grad_norm(of.data(), (int)of.size(), static_cast<double*>(parts.data_ptr()), stream));
      out = py::cast(norm);
    }
    for (size_t i = 0; i < lists.size(); ++i) {
      if (norm.defined()) {
        calls[i].norm_parts = static_cast<const double*>(parts.data_ptr());
        calls[i].n_norm_parts = BNB_GRAD_NORM_PARTS;
        calls[i].max_norm = (float)max_norm.cast<double>();
        calls[i].norm = static_cast<float*>(norm.data_ptr());
      }
      check("bnb_adamw_step", bnb_adamw_step(lists[i].data(), (int)lists[i].size(), &calls[i], stream));
    }
    for (const Tensor* t : changed)
      if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
    return out;
  }

 private:
  struct Entry {
    py::object object, state;            // the parameter; its state's dict, or null
    Tensor p;
    std::vector<py::object> objects;     // the state's tensors, in the order of names_
    std::vector<Tensor> kept;
    int64_t position;
  };

  bool is_of(const py::list& groups, const py::dict& state) const {
    if (groups.size() != groups_.size() || (size_t)PyDict_Size(state.ptr()) != states_.size()) return false;
    PyObject *key, *value;
    size_t k = 0;
    for (Py_ssize_t i = 0; PyDict_Next(state.ptr(), &i, &key, &value); ++k)
      if (key != states_[k].first.ptr() || value != states_[k].second.ptr()) return false;
    for (size_t i = 0; i < groups_.size(); ++i) {
      const py::object params = groups[i]["params"];
      if (!PyList_Check(params.ptr()) || (size_t)PyList_GET_SIZE(params.ptr()) != groups_[i].size()) return false;
      for (size_t j = 0; j < groups_[i].size(); ++j) {
        const Entry& e = groups_[i][j];
        if (PyList_GET_ITEM(params.ptr(), j) != e.object.ptr()) return false;
        if (!e.state.ptr()) {
          if (e.p.grad().defined()) return false;   // its first
          continue;
        }
        for (size_t n = 0; n < names_.size(); ++n)
          if (PyDict_GetItemWithError(e.state.ptr(), keys_[n].ptr()) != e.objects[n].ptr()) return false;
      }
    }
    return true;
  }

  BnbAdamTensor tensor_of(const Entry& e, const Tensor& grad, const c10::Device& dev, std::vector<Tensor>& held, std::vector<const Tensor*>& changed) const {
    const Tensor& p = e.p;
    if (!p.is_cuda()) refuse("AdamW: a parameter is on " + p.device().str() + "; the kernels run on CUDA only (sm_100a) and have no CPU path");
    if (p.device() != dev) refuse("AdamW: parameters on " + p.device().str() + " and " + dev.str() + "; one optimizer serves one device");
    if (grad.layout() != at::kStrided) refuse("AdamW: sparse gradients are not taken");
    if (grad.scalar_type() != p.scalar_type() || grad.sizes() != p.sizes() || grad.device() != dev)
      refuse("AdamW: a gradient has another type, shape or device than its parameter");
    if (!p.is_contiguous() && !p.is_non_overlapping_and_dense())
      throw py::value_error("AdamW: a parameter's elements must lie densely in memory, each in a place of its own");
    BnbAdamTensor t{};
    t.element = element_of("AdamW", p);
    t.n = p.numel();
    t.position = e.position;
    const Tensor &step = e.kept[0], &m = e.kept[1], &v = e.kept[2];
    if (step.scalar_type() != at::kFloat || step.numel() != 1 || step.device() != dev) refuse("AdamW: the state 'step' must be one float32 number on " + dev.str());
    const at::ScalarType type = eight_ ? at::kFloat8_e4m3fn : at::kFloat;
    expect_kept(names_[1], m, p, type, dev);
    expect_kept(names_[2], v, p, type, dev);
    if (eight_) {
      const int64_t blocks = (t.n + STATE_BLOCK - 1) / STATE_BLOCK;
      for (int i : {3, 4}) {
        const Tensor& s = e.kept[i];
        if (s.scalar_type() != at::kFloat || s.dim() != 1 || s.size(0) != blocks || !s.is_contiguous() || s.device() != dev)
          refuse(std::string("AdamW: the state '") + names_[i] + "' must be float32 of shape " + shape_text({blocks}) + ", contiguous, on " + dev.str());
        (i == 3 ? t.m_scale : t.v_scale) = static_cast<float*>(s.data_ptr());
      }
    }
    t.g = grad.data_ptr();
    if (!laid_out_as(grad, p)) {
      held.push_back(at::empty_like(p).copy_(grad));
      t.g = held.back().data_ptr();
    }
    t.p = p.data_ptr();
    t.m = m.data_ptr();
    t.v = v.data_ptr();
    t.step = static_cast<float*>(step.data_ptr());
    changed.push_back(&p);
    for (const Tensor& s : e.kept) changed.push_back(&s);
    return t;
  }

  BnbAdamW call_of(const py::dict& group, uint32_t seed, const Tensor& control, std::vector<Tensor>& held) const {
    BnbAdamW c{};
    c.state_bits = eight_ ? 8 : 32;
    c.seed = seed;
    const py::object lr = group["lr"];
    if (THPVariable_Check(lr.ptr())) {
      const Tensor rate = THPVariable_Unpack(lr.ptr());
      if (rate.numel() != 1) refuse("AdamW: lr must be a number or a tensor of one");
      if (rate.is_cuda()) {
        if (rate.device() != control.device()) refuse("AdamW: lr is on " + rate.device().str() + ", the parameters on " + control.device().str());
        held.push_back(rate.to(at::kFloat));
        c.lr_device = static_cast<const float*>(held.back().data_ptr());
      } else {
        c.lr = rate.item<float>();
      }
    } else {
      c.lr = (float)lr.cast<double>();
    }
    const py::tuple betas = py::tuple(group["betas"]);
    c.beta1 = betas[0].cast<double>();
    c.beta2 = betas[1].cast<double>();
    c.eps = (float)group["eps"].cast<double>();
    c.weight_decay = (float)group["weight_decay"].cast<double>();
    c.control = static_cast<int32_t*>(control.data_ptr());
    return c;
  }

  const bool eight_;
  std::vector<const char*> names_;
  std::vector<py::object> keys_;
  std::vector<std::vector<Entry>> groups_;
  std::vector<std::pair<py::object, py::object>> states_;
};

}  // namespace

void bind_update(py::module& m) {
  m.def("linear_forward", &linear_forward);
  m.def("linear_backward", &linear_backward);
  m.def("linear", torch::wrap_pybind_function(linear));
  py::class_<AdamWPlan>(m, "AdamWPlan").def(py::init<const py::list&, const py::dict&, int>()).def("step", &AdamWPlan::step);
  m.def("policy_loss_forward", &policy_forward);
  m.def("policy_loss_backward", &policy_backward_alone);
  m.def("policy_loss", torch::wrap_pybind_function(policy_loss));
}

}  // namespace host
}  // namespace bnb
