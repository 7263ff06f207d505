// The host side of the operators behind the trunk in an update (yemong/policy_loss.py): checks, outputs and scratch from torch's
// allocator, the launch, the autograd nodes of eager calls.
#include "host_nodes.h"

#include <tuple>

namespace bnb {
namespace host {
namespace {

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

}  // namespace

void bind_update(py::module& m) {
  m.def("policy_loss_forward", &policy_forward);
  m.def("policy_loss_backward", &policy_backward);
  m.def("policy_loss", torch::wrap_pybind_function(policy_loss));
}

}  // namespace host
}  // namespace bnb
