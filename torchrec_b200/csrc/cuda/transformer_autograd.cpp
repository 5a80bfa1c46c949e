// Autograd nodes of the transformer operators in C++.  For the smallest calls - one position scored, one token turned - the kernels take
// a few microseconds and the call is bound by the host: a node here saves the interpreter's share of the forward and the backward
// (a step of 260 rows x 20000 classes x 64 went from 152 to 92 us, a rotation step of 7000 tokens from 131 to 84 us).
#include <ATen/ATen.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/library.h>

#include "transformer_ops.h"

namespace trb {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Gradients of a backward that is itself recorded (create_graph): differentiating them again is an error, not silently zero.  They depend on
// the inputs whether or not the upstream gradient, often the constant one, is recorded too, and the error lies on the way to every input
// (an engine that is asked for one input's gradient walks no other way).
static variable_list once(variable_list grads, const char* name) {
  if (!at::GradMode::is_enabled()) return grads;
  torch::autograd::edge_list inputs;
  for (const auto& edge : torch::autograd::get_current_node()->next_edges())
    if (edge.is_valid()) inputs.push_back(edge);
  auto error = std::make_shared<torch::autograd::Error>(std::string("the gradient of ") + name + " cannot be differentiated again", std::move(inputs));
  for (auto& g : grads)
    if (g.defined()) {
      g = g.detach();
      torch::autograd::set_history(g, error);
    }
  return grads;
}

// A dual tensor need not require a gradient, so that a call without a node would drop its tangent: a derivative of zero.
static void refuse_forward_mode(std::initializer_list<const Tensor*> inputs, const char* name) {
  for (const Tensor* t : inputs) TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(), name, " has no forward-mode derivative on CUDA");
}

static c10::optional<Tensor> opt(const Tensor& t) { return t.defined() ? c10::optional<Tensor>(t) : c10::nullopt; }

// ---- softmax over the whole catalogue ---------------------------------------------------------------------
// the weight as the kernel reads it: bf16 rows on 16-byte boundaries, zero columns up to a multiple of 8
static Tensor kernel_rows(const Tensor& weight, const c10::optional<Tensor>& rounded) {
  Tensor w = rounded.has_value() && rounded->defined() ? *rounded : weight;
  if (w.scalar_type() != at::kBFloat16) w = w.to(at::kBFloat16);
  if (w.size(1) % 8) return at::constant_pad_nd(w, {0, (8 - w.size(1) % 8) % 8});
  if (w.stride(1) != 1 || w.stride(0) % 8 || w.stride(0) < w.size(1) || reinterpret_cast<uintptr_t>(w.data_ptr()) % 16) w = w.clone(at::MemoryFormat::Contiguous);
  return w;
}

struct FullSoftmaxLoss : public torch::autograd::Function<FullSoftmaxLoss> {
  static Tensor forward(AutogradContext* ctx, const Tensor& h, const Tensor& weight, const c10::optional<Tensor>& bias, const Tensor& targets,
                        const c10::optional<Tensor>& rounded, int64_t ignore_index, int64_t reduction, int64_t grad) {
    const Tensor w = kernel_rows(weight, rounded);
    auto [loss, state] = full_softmax_fwd(h, w, targets, bias, ignore_index, reduction, grad, 0);
    if (grad > 0) {
      // the caller's weight is saved too where the kernel read a copy, so that a change in place is noticed
      ctx->save_for_backward({state, weight, w.is_same(weight) ? Tensor() : w});
      ctx->saved_data["shape"] = std::vector<int64_t>{h.size(0), h.size(1), reduction, grad};
      const bool has_bias = bias.has_value() && bias->defined();
      ctx->saved_data["types"] = std::vector<int64_t>{h.scalar_type() == at::kFloat, weight.scalar_type() == at::kFloat, has_bias, has_bias && bias->scalar_type() == at::kFloat};
    }
    return loss;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const auto shape = ctx->saved_data["shape"].toIntVector(), types = ctx->saved_data["types"].toIntVector();
    const Tensor& w = saved[2].defined() ? saved[2] : saved[1];
    const int64_t D = shape[1];
    const bool has_bias = types[2] != 0;
    const bool want_h = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1), want_b = has_bias && ctx->needs_input_grad(2);
    Tensor dh, dw, db;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      std::tie(dh, dw, db) = full_softmax_bwd(grads[0], w, saved[0], shape[0], D, has_bias, shape[2], shape[3] == 2, want_h, want_w, want_b, types[0] != 0, types[1] != 0, types[3] != 0);
      if (want_w && dw.size(1) != D) dw = dw.narrow(1, 0, D).contiguous();
    }
    variable_list out(8);
    if (want_h) out[0] = dh;
    if (want_w) out[1] = dw;
    if (want_b) out[2] = db;
    return once(std::move(out), "full_softmax_loss");
  }
};

static void check_full_softmax(const Tensor& h, const Tensor& weight, const c10::optional<Tensor>& bias, const Tensor& targets) {
  TORCH_CHECK_VALUE(h.dim() == 2 && weight.dim() == 2 && h.size(1) == weight.size(1) && weight.size(0) > 0 && h.size(1) > 0,
                    "full_softmax_loss: h [P, D] and weight [V, D] with V, D > 0, got ", h.sizes(), " and ", weight.sizes());
  TORCH_CHECK_VALUE(targets.dim() == 1 && targets.size(0) == h.size(0) && (targets.scalar_type() == at::kLong || targets.scalar_type() == at::kInt),
                    "full_softmax_loss: targets is an int32 or int64 [P], got ", targets.scalar_type(), " ", targets.sizes());
  if (bias.has_value() && bias->defined()) {
    TORCH_CHECK_VALUE(bias->dim() == 1 && bias->size(0) == weight.size(0), "full_softmax_loss: bias is [V], got ", bias->sizes(), " for ", weight.size(0), " classes");
    TORCH_CHECK_VALUE(bias->device() == h.device(), "full_softmax_loss: bias is on ", bias->device(), ", h on ", h.device());
  }
  TORCH_CHECK_VALUE(weight.device() == h.device(), "full_softmax_loss: weight is on ", weight.device(), ", h on ", h.device());
  TORCH_CHECK_VALUE(targets.device() == h.device(), "full_softmax_loss: targets is on ", targets.device(), ", h on ", h.device());
}

static Tensor full_softmax_loss_plain(const Tensor& h, const Tensor& weight, const c10::optional<Tensor>& bias, const Tensor& targets, const c10::optional<Tensor>& rounded,
                                      int64_t ignore_index, int64_t reduction) {
  check_full_softmax(h, weight, bias, targets);
  return std::get<0>(full_softmax_fwd(h, kernel_rows(weight, rounded), targets, bias, ignore_index, reduction, 0, 0));
}

static Tensor full_softmax_loss_autograd(const Tensor& h, const Tensor& weight, const c10::optional<Tensor>& bias, const Tensor& targets, const c10::optional<Tensor>& rounded,
                                         int64_t ignore_index, int64_t reduction) {
  const Tensor b = bias.value_or(Tensor());
  refuse_forward_mode({&h, &weight, &b}, "full_softmax_loss");
  int64_t grad = 0;
  if (at::GradMode::is_enabled()) grad = h.requires_grad() ? 2 : int64_t(weight.requires_grad() || (b.defined() && b.requires_grad()));
  if (grad == 0) {  // no node
    at::AutoDispatchBelowADInplaceOrView below;
    return full_softmax_loss_plain(h, weight, bias, targets, rounded, ignore_index, reduction);
  }
  check_full_softmax(h, weight, bias, targets);
  return FullSoftmaxLoss::apply(h, weight, bias, targets, rounded, ignore_index, reduction, grad);
}

// ---- norm and rotation of queries and keys ------------------------------------------------------------------
// contiguous rows that start on 16-byte boundaries
static Tensor rows16(const Tensor& t) {
  if (t.stride(1) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && (t.stride(0) * t.element_size()) % 16 == 0 && (t.size(0) <= 1 || t.stride(0) >= t.size(1))) return t;
  return t.clone(at::MemoryFormat::Contiguous);
}
static c10::optional<Tensor> fp32(const c10::optional<Tensor>& w) {
  return w.has_value() && w->defined() ? c10::optional<Tensor>(w->to(at::kFloat).contiguous()) : c10::nullopt;
}

struct QKNormRotary : public torch::autograd::Function<QKNormRotary> {
  static Tensor forward(AutogradContext* ctx, const Tensor& qkv_in, const c10::optional<Tensor>& qw_in, const c10::optional<Tensor>& kw_in, const Tensor& positions,
                        const Tensor& inv_freq, at::IntArrayRef sections, int64_t heads, int64_t kv_heads, double eps, bool norm, bool interleaved) {
    const Tensor qkv = rows16(qkv_in);
    const auto qw = fp32(qw_in), kw = fp32(kw_in);
    Tensor out = qk_norm_rotary_fwd(qkv, positions, inv_freq, qw, kw, sections, heads, kv_heads, eps, norm, interleaved);
    // the callers' tensors are saved next to copies of them, so that a change in place is noticed
    ctx->save_for_backward({qkv, positions, inv_freq, qw.value_or(Tensor()), kw.value_or(Tensor()), qkv.is_same(qkv_in) ? Tensor() : qkv_in,
                            qw && !qw->is_same(*qw_in) ? *qw_in : Tensor(), kw && !kw->is_same(*kw_in) ? *kw_in : Tensor()});
    std::vector<int64_t> ints{heads, kv_heads, norm, interleaved, qw ? int64_t(qw_in->scalar_type()) : 0, kw ? int64_t(kw_in->scalar_type()) : 0};
    ints.insert(ints.end(), sections.begin(), sections.end());
    ctx->saved_data["ints"] = ints;
    ctx->saved_data["eps"] = eps;
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const auto ints = ctx->saved_data["ints"].toIntVector();
    // needs_input_grad counts the tensors that were passed
    const bool want_q = saved[3].defined() && ctx->needs_input_grad(1), want_k = saved[4].defined() && ctx->needs_input_grad(saved[3].defined() ? 2 : 1);
    Tensor dqkv, dw;
    variable_list out(11);
    {
      at::AutoDispatchBelowADInplaceOrView below;
      std::tie(dqkv, dw) = qk_norm_rotary_bwd(rows16(grads[0]), saved[0], saved[1], saved[2], opt(saved[3]), opt(saved[4]), at::IntArrayRef(ints).slice(6), ints[0], ints[1],
                                              ctx->saved_data["eps"].toDouble(), ints[2] != 0, ints[3] != 0, want_q || want_k);
      if (want_q) out[1] = dw.select(0, 0).to(at::ScalarType(ints[4]));
      if (want_k) out[2] = dw.select(0, 1).to(at::ScalarType(ints[5]));
    }
    if (ctx->needs_input_grad(0)) out[0] = dqkv;
    return once(std::move(out), "qk_norm_rotary");
  }
};

static Tensor check_rotary(const Tensor& qkv, const c10::optional<Tensor>& qw, const c10::optional<Tensor>& kw, const Tensor& positions, const Tensor& inv_freq,
                           at::IntArrayRef sections, int64_t heads, int64_t kv_heads, double eps) {
  TORCH_CHECK_VALUE(heads >= 1 && kv_heads >= 1 && qkv.dim() == 2 && qkv.size(1) > 0 && qkv.size(1) % (heads + 2 * kv_heads) == 0,
                    "qk_norm_rotary: qkv is [T, (heads + 2 kv_heads) * head_dim], got ", qkv.sizes(), " for ", heads, " and ", kv_heads, " heads");
  const int64_t T = qkv.size(0), dim = qkv.size(1) / (heads + 2 * kv_heads), axes = int64_t(sections.size());
  TORCH_CHECK_VALUE(inv_freq.dim() == 1 && inv_freq.is_floating_point() && inv_freq.size(0) >= 1 && inv_freq.size(0) <= dim / 2,
                    "qk_norm_rotary: inv_freq holds 1 to head_dim / 2 = ", dim / 2, " frequencies, got ", inv_freq.scalar_type(), " ", inv_freq.sizes());
  const bool one = positions.dim() == 1 && axes == 1 && positions.size(0) == T, many = positions.dim() == 2 && positions.size(0) == axes && positions.size(1) == T;
  TORCH_CHECK_VALUE((positions.scalar_type() == at::kLong || positions.scalar_type() == at::kInt) && (one || many),
                    "qk_norm_rotary: positions is an int32 or int64 [T] or [axes, T], got ", positions.scalar_type(), " ", positions.sizes(), " for ", T, " tokens and ", axes,
                    " axes");
  int64_t sum = 0;
  bool negative = false;
  for (const auto n : sections) {
    sum += n;
    negative = negative || n < 0;
  }
  TORCH_CHECK_VALUE(axes >= 1 && axes <= 8 && !negative && sum == inv_freq.size(0), "qk_norm_rotary: up to 8 sections that add up to the ", inv_freq.size(0),
                    " frequencies, got ", sections);
  for (const auto* w : {&qw, &kw})
    if (w->has_value() && (*w)->defined()) {
      TORCH_CHECK_VALUE((*w)->dim() == 1 && (*w)->size(0) == dim && (*w)->is_floating_point(), "qk_norm_rotary: ", w == &qw ? "q_weight" : "k_weight", " is [head_dim] = [", dim,
                        "], got ", (*w)->scalar_type(), " ", (*w)->sizes());
      TORCH_CHECK_VALUE((*w)->device() == qkv.device(), "qk_norm_rotary: ", w == &qw ? "q_weight" : "k_weight", " is on ", (*w)->device(), ", qkv on ", qkv.device());
    }
  TORCH_CHECK_VALUE(positions.device() == qkv.device(), "qk_norm_rotary: positions is on ", positions.device(), ", qkv on ", qkv.device());
  TORCH_CHECK_VALUE(inv_freq.device() == qkv.device(), "qk_norm_rotary: inv_freq is on ", inv_freq.device(), ", qkv on ", qkv.device());
  TORCH_CHECK_VALUE(eps >= 0, "qk_norm_rotary: eps is not negative, got ", eps);
  return one ? positions.unsqueeze(0) : positions;
}

static Tensor frequencies(const Tensor& f) { return f.detach().to(at::kDouble).contiguous(); }

static Tensor qk_norm_rotary_plain(const Tensor& qkv, const Tensor& positions, const Tensor& inv_freq, const c10::optional<Tensor>& qw, const c10::optional<Tensor>& kw,
                                   at::IntArrayRef sections, int64_t heads, int64_t kv_heads, double eps, bool norm, bool interleaved) {
  const Tensor pos = check_rotary(qkv, qw, kw, positions, inv_freq, sections, heads, kv_heads, eps);
  return qk_norm_rotary_fwd(rows16(qkv), pos, frequencies(inv_freq), fp32(qw), fp32(kw), sections, heads, kv_heads, eps, norm, interleaved);
}

static Tensor qk_norm_rotary_autograd(const Tensor& qkv, const Tensor& positions, const Tensor& inv_freq, const c10::optional<Tensor>& qw, const c10::optional<Tensor>& kw,
                                      at::IntArrayRef sections, int64_t heads, int64_t kv_heads, double eps, bool norm, bool interleaved) {
  const Tensor q = qw.value_or(Tensor()), k = kw.value_or(Tensor());
  refuse_forward_mode({&qkv, &q, &k}, "qk_norm_rotary");
  auto wants = [](const Tensor& t) { return t.defined() && t.requires_grad(); };
  if (!at::GradMode::is_enabled() || !(qkv.requires_grad() || wants(q) || wants(k))) {  // no node
    at::AutoDispatchBelowADInplaceOrView below;
    return qk_norm_rotary_plain(qkv, positions, inv_freq, qw, kw, sections, heads, kv_heads, eps, norm, interleaved);
  }
  const Tensor pos = check_rotary(qkv, qw, kw, positions, inv_freq, sections, heads, kv_heads, eps);
  return QKNormRotary::apply(qkv, qw, kw, pos, frequencies(inv_freq), sections, heads, kv_heads, eps, norm, interleaved);
}

}  // namespace trb

TORCH_LIBRARY_FRAGMENT(trb200, m) {
  m.def("full_softmax_loss(Tensor h, Tensor weight, Tensor? bias, Tensor targets, Tensor? rounded, int ignore_index, int reduction) -> Tensor");
  m.def("qk_norm_rotary(Tensor qkv, Tensor positions, Tensor inv_freq, Tensor? q_weight, Tensor? k_weight, int[] sections, int heads, int kv_heads, float eps, bool norm, "
        "bool interleaved) -> Tensor");
}

TORCH_LIBRARY_IMPL(trb200, AutogradCUDA, m) {
  m.impl("full_softmax_loss", &trb::full_softmax_loss_autograd);
  m.impl("qk_norm_rotary", &trb::qk_norm_rotary_autograd);
}

TORCH_LIBRARY_IMPL(trb200, CUDA, m) {
  m.impl("full_softmax_loss", &trb::full_softmax_loss_plain);
  m.impl("qk_norm_rotary", &trb::qk_norm_rotary_plain);
}
