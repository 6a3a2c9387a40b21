// Autograd nodes of the operators around a training step's products (layer norm, rotary positions) and the registration of these and of the
// gradient norm.  The nodes are C++: a node written in Python costs 10 to 20 us per pass, more than the kernels of a short sequence.
#include <ATen/ATen.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include "host.h"

namespace q38 {
// vocab_loss.cu
std::vector<at::Tensor> vocab_loss_fwd(const at::Tensor& hidden, const at::Tensor& weight, const at::Tensor& target, int64_t reduction, const at::Tensor& err);
std::vector<at::Tensor> vocab_loss_bwd(const at::Tensor& g, const at::Tensor& hidden, const at::Tensor& weight, const at::Tensor& target, const at::Tensor& lse2, const at::Tensor& count,
                                       int64_t reduction, bool want_dh, bool fp32_dh, bool want_dw, bool fp32_dw, const c10::optional<at::Tensor>& grad, int64_t workspace,
                                       const at::Tensor& err);

namespace {

using at::Tensor;
using OptTensor = c10::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

OptTensor optional_of(const Tensor& t) { return t.defined() ? OptTensor(t) : c10::nullopt; }
bool wants_grad(const OptTensor& t) { return t.has_value() && t->requires_grad(); }

// ---- layer norm ---------------------------------------------------------------------------------------------------------------
// [rows, dim] with contiguous columns and one distance between rows, without a copy where x has that already
Tensor as_rows(const Tensor& x) {
  const auto r = x.reshape({-1, x.size(-1)});
  return r.stride(1) == 1 || r.size(1) == 1 ? r : r.contiguous();
}

struct LayerNorm : public torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& w, const OptTensor& b, double eps, at::ScalarType out_type) {
    auto out = layer_norm_fwd(as_rows(x), w, b, eps, out_type, true);
    ctx->save_for_backward({x, w.value_or(Tensor()), b.value_or(Tensor()), out[1], out[2]});
    return out[0].view(x.sizes());
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "layer_norm: a gradient of the gradient is not available");
    auto saved = ctx->get_saved_variables();
    const OptTensor w = optional_of(saved[1]), b = optional_of(saved[2]);
    const size_t b_edge = w.has_value() ? 2 : 1;                   // edges are counted over the tensors that were given
    auto out = layer_norm_bwd(as_rows(grads[0]), as_rows(saved[0]), w, b, saved[3], saved[4], ctx->needs_input_grad(0), w.has_value() && ctx->needs_input_grad(1),
                              b.has_value() && ctx->needs_input_grad(b_edge));
    return {out[0].defined() ? out[0].view(saved[0].sizes()) : out[0], out[1], out[2], Tensor(), Tensor()};
  }
};

Tensor layer_norm(const Tensor& x, const OptTensor& w, const OptTensor& b, double eps, c10::optional<at::ScalarType> out_type) {
  TORCH_CHECK(x.dim() > 0 && x.size(-1) > 0, "layer_norm: an input with a last dimension that is not empty required");
  const at::ScalarType to = out_type.value_or(x.scalar_type());
  if (at::GradMode::is_enabled() && (x.requires_grad() || wants_grad(w) || wants_grad(b))) return LayerNorm::apply(x, w, b, eps, to);
  return layer_norm_fwd(as_rows(x), w, b, eps, to, false)[0].view(x.sizes());
}

// ---- rotary positions ------------------------------------------------------------------------------------------------------------
struct Rotary : public torch::autograd::Function<Rotary> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const OptTensor& k, const Tensor& pos, const Tensor& freq, double magnitude, bool interleaved) {
    auto [qo, ko] = rotary_apply(q, k.value_or(Tensor()), pos, freq, magnitude, interleaved, 1.0);
    ctx->save_for_backward({pos, freq});
    ctx->saved_data["magnitude"] = magnitude;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->set_materialize_grads(false);
    return k.has_value() ? variable_list{qo, ko} : variable_list{qo};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "rotary: a gradient of the gradient is not available");
    auto saved = ctx->get_saved_variables();
    const bool keys = grads.size() > 1;
    const Tensor dq = grads[0].defined() && ctx->needs_input_grad(0) ? grads[0] : Tensor();
    const Tensor dk = keys && grads[1].defined() && ctx->needs_input_grad(1) ? grads[1] : Tensor();
    std::pair<Tensor, Tensor> out;
    if (dq.defined() || dk.defined()) out = rotary_apply(dq, dk, saved[0], saved[1], ctx->saved_data["magnitude"].toDouble(), ctx->saved_data["interleaved"].toBool(), -1.0);
    return {out.first, out.second, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

std::vector<Tensor> rotary(const Tensor& q, const OptTensor& k, const Tensor& pos, const Tensor& freq, double magnitude, bool interleaved) {
  rotary_check(q, k, pos, freq);
  if (at::GradMode::is_enabled() && (q.requires_grad() || wants_grad(k))) return Rotary::apply(q, k, pos, freq, magnitude, interleaved);
  auto [qo, ko] = rotary_apply(q, k.value_or(Tensor()), pos, freq, magnitude, interleaved, 1.0);
  return k.has_value() ? std::vector<Tensor>{qo, ko} : std::vector<Tensor>{qo};
}

}  // namespace
}  // namespace q38

TORCH_LIBRARY_FRAGMENT(q38, m) {
  m.def("layer_norm(Tensor x, Tensor? w, Tensor? b, float eps, ScalarType? out_dtype=None) -> Tensor", &q38::layer_norm);
  m.def("rotary(Tensor q, Tensor? k, Tensor positions, Tensor frequencies, float magnitude, bool interleaved) -> Tensor[]", &q38::rotary);
  m.def("vocab_loss_fwd(Tensor hidden, Tensor weight, Tensor target, int reduction, Tensor(a!) err) -> Tensor[]", &q38::vocab_loss_fwd);
  m.def("vocab_loss_bwd(Tensor g, Tensor hidden, Tensor weight, Tensor target, Tensor lse2, Tensor count, int reduction, bool want_dh, bool fp32_dh, bool want_dw, bool fp32_dw, "
        "Tensor(b!)? grad, int workspace, Tensor(a!) err) -> Tensor[]", &q38::vocab_loss_bwd);
  m.def("grad_norm(Tensor[] grads) -> Tensor", [](at::TensorList g) { return q38::clip_grad_norm(g, {}, 1.0, false); });
  m.def("clip_grad_norm_(Tensor(a!)[] grads, float max_norm) -> Tensor", [](at::TensorList g, double m) { return q38::clip_grad_norm(g, {}, m, true); });
  m.def("clip_grad_norm_out(Tensor[] grads, Tensor(a!)[] out, float max_norm) -> Tensor", [](at::TensorList g, at::TensorList o, double m) { return q38::clip_grad_norm(g, o, m, true); });
}
