// Autograd nodes of the operators around a training step's products, and their registration.  The nodes are written out in C++: one in Python costs 10 to 20 us
// per pass, torch's own wrapper for C++ functions half of that, and the kernels of a short sequence take 2 to 5.
#include <ATen/ATen.h>
#include <c10/core/DispatchKeySet.h>
#include <c10/core/InferenceMode.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/library.h>

#include "training.h"

namespace q38 {
namespace {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

// Gradients enabled inside inference mode are not recorded
bool recording() { return at::GradMode::is_enabled() && !c10::InferenceMode::is_enabled(); }
bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }
OptTensor optional_of(const Tensor& t) { return t.defined() ? OptTensor(t) : c10::nullopt; }

// The entries are registered for every kind of tensor, and the kernels take addresses: a fake or wrapped tensor has a null one (a launch would fault), a batched or
// transformed one none of its own.  A tensor with a tangent (forward mode) would give a result without one, which counts as a constant.
void check_operand(const char* name, const Tensor& t) {
  constexpr c10::DispatchKeySet without{c10::DispatchKey::Python, c10::DispatchKey::Functionalize, c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::Batched, c10::DispatchKey::FuncTorchGradWrapper,
                                        c10::DispatchKey::ZeroTensor};
  TORCH_CHECK_VALUE(!t.defined() || !t.key_set().has_any(without), name, ": a tensor with values in memory of its own is required, not one that is fake, wrapped, batched or transformed");
  TORCH_CHECK(!t.defined() || !t._fw_grad(0).defined(), name, ": derivatives in forward mode are not available");
}
void check_operand(const char* name, const OptTensor& t) { if (t.has_value()) check_operand(name, *t); }
void check_operand(const char* name, at::TensorList list) { for (const Tensor& t : list) check_operand(name, t); }

// A negated view (the imaginary part of a conjugate) holds its values with the other sign: they are written out.
Tensor values(const Tensor& t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }
Tensor values(const OptTensor& t) { return t.has_value() ? values(*t) : Tensor(); }

void first_order_only(const char* name) { TORCH_CHECK(!at::GradMode::is_enabled(), name, ": a gradient of the gradient is not available"); }

// ---- layer norm ---------------------------------------------------------------------------------------------------------------
struct LayerNormBackward : public Node {
  SavedVariable x, w;
  Tensor stats;
  OptTensor b;                     // of the bias only its type and length count: a detached alias, so that changing it is allowed
  std::string name() const override { return "Q38LayerNormBackward"; }
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    x.reset_data(); w.reset_data(); stats.reset();
  }
  variable_list apply(variable_list&& grads) override {
    const std::lock_guard<std::mutex> lock(mutex_);
    first_order_only("layer_norm");
    if (!grads[0].defined()) return variable_list(3);
    check_operand("layer_norm", grads[0]);
    auto self = shared_from_this();
    const Tensor xs = x.unpack(self), ws = w.unpack(self);
    auto out = layer_norm_bwd(values(grads[0]), xs, optional_of(ws), b, stats, task_should_compute_output(0), ws.defined() && task_should_compute_output(1),
                              b.has_value() && task_should_compute_output(2));
    return {out[0], out[1], out[2]};
  }
};

Tensor layer_norm(const Tensor& x_, const OptTensor& w, const OptTensor& b, double eps, c10::optional<at::ScalarType> out_type) {
  check_operand("layer_norm", x_);
  check_operand("layer_norm", w);
  check_operand("layer_norm", b);
  const Tensor x = values(x_), wt = values(w), bt = values(b);
  const bool grad = recording() && (wants_grad(x) || wants_grad(wt) || wants_grad(bt));
  Tensor y, stats;
  {
    const at::NoGradGuard none;
    std::tie(y, stats) = layer_norm_fwd(x, optional_of(wt), optional_of(bt), eps, out_type.value_or(x.scalar_type()), grad);
  }
  if (grad) {
    auto node = std::shared_ptr<LayerNormBackward>(new LayerNormBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x, wt, bt));
    node->x = SavedVariable(x, false);
    node->w = SavedVariable(wt, false);
    node->stats = stats;
    if (bt.defined()) node->b = bt.detach();
    torch::autograd::set_history(y, node);
  }
  return y;
}

// ---- rotary positions ------------------------------------------------------------------------------------------------------------
struct RotaryBackward : public Node {
  SavedVariable pos, freq;
  double magnitude;
  bool interleaved;
  std::string name() const override { return "Q38RotaryBackward"; }
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    pos.reset_data(); freq.reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    const std::lock_guard<std::mutex> lock(mutex_);
    first_order_only("rotary");
    const Tensor dq = task_should_compute_output(0) ? values(grads[0]) : Tensor(), dk = grads.size() > 1 && task_should_compute_output(1) ? values(grads[1]) : Tensor();
    if (!dq.defined() && !dk.defined()) return variable_list(2);
    check_operand("rotary", grads);
    auto out = rotary_apply(dq, dk, pos.unpack(), freq.unpack(), magnitude, interleaved, -1.0);
    return {out.first, out.second};
  }
};

std::vector<Tensor> rotary(const Tensor& q_, const OptTensor& k, const Tensor& pos_, const Tensor& frequencies, double magnitude, bool interleaved) {
  for (const Tensor* t : {&q_, &pos_, &frequencies}) check_operand("rotary", *t);
  check_operand("rotary", k);
  TORCH_CHECK_VALUE(!(recording() && frequencies.requires_grad()), "rotary: a gradient of the frequencies is not available; detached ones are required");
  const Tensor q = values(q_), kt = values(k), pos = values(pos_), signed_freq = values(frequencies), freq = signed_freq.is_contiguous() ? signed_freq : signed_freq.contiguous();
  rotary_check(q, optional_of(kt), pos, freq);
  const bool grad = recording() && (wants_grad(q) || wants_grad(kt));
  std::pair<Tensor, Tensor> out;
  {
    const at::NoGradGuard none;                                    // layouts that need a copy
    out = rotary_apply(q, kt, pos, freq, magnitude, interleaved, 1.0);
  }
  if (grad) {
    auto node = std::shared_ptr<RotaryBackward>(new RotaryBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(q, kt));
    node->pos = SavedVariable(pos, false);
    node->freq = SavedVariable(freq, false);
    node->magnitude = magnitude;
    node->interleaved = interleaved;
    torch::autograd::set_history(out.first, node);
    if (k.has_value()) torch::autograd::set_history(out.second, node);
  }
  return k.has_value() ? std::vector<Tensor>{out.first, out.second} : std::vector<Tensor>{out.first};
}

// ---- vocabulary loss ---------------------------------------------------------------------------------------------------------------
struct VocabLossBackward : public Node {
  SavedVariable hidden, weight, target;      // [rows, h], [vocabulary, h] in bf16 and [rows], as the products take them
  Tensor lse2, count, err, parameter;        // parameter: of the trainer's arena, its gradient buffer is added to
  std::vector<int64_t> shape;                // of the hidden states as they were given
  int64_t reduction, workspace;
  bool fp32_dh, fp32_dw;
  std::string name() const override { return "Q38VocabLossBackward"; }
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    hidden.reset_data(); weight.reset_data(); target.reset_data();
    lse2.reset(); count.reset(); parameter.reset();
  }
  variable_list apply(variable_list&& grads) override {
    const std::lock_guard<std::mutex> lock(mutex_);
    first_order_only("vocabulary_cross_entropy");
    if (!grads[0].defined()) return variable_list(2);
    check_operand("vocabulary_cross_entropy", grads[0]);
    const Tensor h = hidden.unpack(), w = weight.unpack(), t = target.unpack();
    const Tensor given = values(grads[0]), g = given.scalar_type() == at::kFloat && given.is_contiguous() ? given : given.to(at::kFloat).contiguous();
    const bool want_dw = task_should_compute_output(1);
    Tensor buffer;
    if (want_dw && parameter.defined()) {
      const Tensor& own = parameter.grad();
      if (own.defined() && own.scalar_type() == at::kFloat && own.is_contiguous() && own.size(1) % 4 == 0 && (reinterpret_cast<uintptr_t>(own.data_ptr()) & 15) == 0) buffer = own;
    }
    auto out = vocab_loss_bwd(g, h, w, t, lse2, count, reduction, task_should_compute_output(0), fp32_dh, want_dw, fp32_dw, buffer, workspace, err);
    return {out.first.defined() && shape.size() != 2 ? out.first.view(shape) : out.first, out.second};
  }
};

// hidden [..., h]; weight [vocabulary, h] and the same in bf16; target of hidden's leading shape.
Tensor vocab_loss(const Tensor& hidden_, const Tensor& weight, const Tensor& weight16, const Tensor& target_, int64_t reduction, bool managed, int64_t workspace, const Tensor& err) {
  for (const Tensor* t : {&hidden_, &weight, &weight16, &target_, &err}) check_operand("vocabulary_cross_entropy", *t);
  const Tensor hidden = values(hidden_), target = values(target_);
  TORCH_CHECK_VALUE(weight.dim() == 2 && hidden.dim() >= 1 && hidden.size(-1) == weight.size(1) && weight.numel() > 0,
                    "vocabulary_cross_entropy: hidden [..., h] and weight [vocabulary, h] required");
  TORCH_CHECK_VALUE(target.sizes() == hidden.sizes().slice(0, hidden.dim() - 1) && target.scalar_type() == at::kLong, "vocabulary_cross_entropy: int64 targets of hidden's leading shape required");
  for (const Tensor* t : {&hidden, &weight})
    TORCH_CHECK_VALUE(t->scalar_type() == at::kBFloat16 || t->scalar_type() == at::kFloat, "vocabulary_cross_entropy: bf16 or fp32 hidden states and weight required");
  TORCH_CHECK_VALUE(hidden.is_cuda() && weight.device() == hidden.device() && target.device() == hidden.device(), "vocabulary_cross_entropy: hidden, weight and target on one device required");
  const bool grad = recording() && (wants_grad(hidden) || wants_grad(weight));
  Tensor h, w, t, loss, lse2, count;
  {
    const at::NoGradGuard none;
    // Views of what was given where nothing has to be converted or copied: a change before the backward is then noticed.  Copies into padded rows are kept for it.
    h = hidden.scalar_type() == at::kBFloat16 ? hidden : hidden.to(at::kBFloat16);
    h = vocab_rows(h.dim() == 2 ? h : h.reshape({-1, h.size(-1)}));
    w = vocab_rows(values(weight16));
    t = target.dim() == 1 ? target : target.reshape({-1});
    if (!t.is_contiguous()) t = t.contiguous();
    auto out = vocab_loss_fwd(h, w, t, target.sizes(), reduction, err);
    loss = out[0]; lse2 = out[1]; count = out[2];
  }
  if (grad) {
    auto node = std::shared_ptr<VocabLossBackward>(new VocabLossBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(hidden, weight));
    node->hidden = SavedVariable(h, false);
    node->weight = SavedVariable(w, false);
    node->target = SavedVariable(t, false);
    node->lse2 = lse2; node->count = count; node->err = err;
    if (managed) node->parameter = weight;
    node->shape = hidden.sizes().vec();
    node->reduction = reduction; node->workspace = workspace;
    node->fp32_dh = hidden.scalar_type() == at::kFloat; node->fp32_dw = weight.scalar_type() == at::kFloat;
    torch::autograd::set_history(loss, node);
  }
  return loss;
}

Tensor clip(const char* name, at::TensorList grads, at::TensorList outs, double max_norm, bool scale) {
  check_operand(name, grads);
  check_operand(name, outs);
  // the norm and the scaling in place are the same for either sign; a result of the other sign takes its gradient's values with that sign
  const at::NoGradGuard none;
  std::vector<Tensor> turned;
  for (size_t i = 0; i < outs.size() && i < grads.size(); ++i)
    if (outs[i].is_neg() != grads[i].is_neg()) {
      if (turned.empty()) turned = grads.vec();
      turned[i] = outs[i].is_neg() ? grads[i].neg() : grads[i].resolve_neg();
    }
  return clip_grad_norm(turned.empty() ? grads : at::TensorList(turned), outs, max_norm, scale);
}

}  // namespace
}  // namespace q38

TORCH_LIBRARY_FRAGMENT(q38, m) {
  m.def("layer_norm(Tensor x, Tensor? w, Tensor? b, float eps, ScalarType? out_dtype=None) -> Tensor", &q38::layer_norm);
  m.def("rotary(Tensor q, Tensor? k, Tensor positions, Tensor frequencies, float magnitude, bool interleaved) -> Tensor[]", &q38::rotary);
  m.def("vocab_loss(Tensor hidden, Tensor weight, Tensor weight16, Tensor target, int reduction, bool managed, int workspace, Tensor(a!) err) -> Tensor", &q38::vocab_loss);
  m.def("grad_norm(Tensor[] grads) -> Tensor", [](at::TensorList g) { return q38::clip("grad_norm", g, {}, 1.0, false); });
  m.def("clip_grad_norm_(Tensor(a!)[] grads, float max_norm) -> Tensor", [](at::TensorList g, double m) { return q38::clip("clip_grad_norm", g, {}, m, true); });
  m.def("clip_grad_norm_out(Tensor[] grads, Tensor(a!)[] out, float max_norm) -> Tensor",
        [](at::TensorList g, at::TensorList o, double m) { return q38::clip("clip_grad_norm", g, o, m, true); });
  m.def("check_operands(Tensor[] tensors, str name) -> ()", [](at::TensorList t, c10::string_view name) { q38::check_operand(std::string(name).c_str(), t); });
}
