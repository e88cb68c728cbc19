// Autograd of the LM head's cross entropy (an additive operator of this build;
// the other operators have no gradient, as in the reference).
#include <ATen/core/dispatch/Dispatcher.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include "cid_engine/ops.hpp"

namespace cid::engine {
namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Pair = std::tuple<at::Tensor, at::Tensor>;

Pair call_forward(const at::Tensor& labels, const at::Tensor& hidden, const at::Tensor& weight,
                  std::int64_t ignore) {
  static const auto op =
      c10::Dispatcher::singleton()
          .findSchemaOrThrow("cid_engine::lm_head_cross_entropy", "")
          .typed<Pair(const at::Tensor&, const at::Tensor&, const at::Tensor&, std::int64_t)>();
  return op.call(labels, hidden, weight, ignore);
}

Pair call_backward(const std::optional<at::Tensor>& gl, const std::optional<at::Tensor>& ge,
                   const at::Tensor& labels, const at::Tensor& hidden, const at::Tensor& weight,
                   const at::Tensor& lse, std::int64_t ignore, bool need_hidden,
                   bool need_weight) {
  static const auto op =
      c10::Dispatcher::singleton()
          .findSchemaOrThrow("cid_engine::lm_head_cross_entropy_backward", "")
          .typed<Pair(const std::optional<at::Tensor>&, const std::optional<at::Tensor>&,
                      const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                      std::int64_t, bool, bool)>();
  return op.call(gl, ge, labels, hidden, weight, lse, ignore, need_hidden, need_weight);
}

struct HeadLoss : torch::autograd::Function<HeadLoss> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& labels,
                               const at::Tensor& hidden, const at::Tensor& weight,
                               std::int64_t ignore) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [loss, lse] = call_forward(labels, hidden, weight, ignore);
    ctx->set_materialize_grads(false);
    ctx->saved_data["ignore"] = ignore;
    ctx->save_for_backward({labels, hidden, weight, lse});
    return {loss, lse};
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const bool need_hidden = ctx->needs_input_grad(1), need_weight = ctx->needs_input_grad(2);
    if (!grads[0].defined() && !grads[1].defined()) return variable_list(4);
    const auto saved = ctx->get_saved_variables();
    auto optional = [](const at::Tensor& t) {
      return t.defined() ? std::optional<at::Tensor>(t) : std::nullopt;
    };
    auto [gh, gw] = call_backward(optional(grads[0]), optional(grads[1]), saved[0], saved[1],
                                  saved[2], saved[3], ctx->saved_data["ignore"].toInt(),
                                  need_hidden, need_weight);
    return {at::Tensor(), need_hidden ? gh : at::Tensor(), need_weight ? gw : at::Tensor(),
            at::Tensor()};
  }
};

// The gradient as an autograd node whose own gradient is refused.
struct HeadLossBackward : torch::autograd::Function<HeadLossBackward> {
  static variable_list forward(AutogradContext*, const std::optional<at::Tensor>& gl,
                               const std::optional<at::Tensor>& ge, const at::Tensor& labels,
                               const at::Tensor& hidden, const at::Tensor& weight,
                               const at::Tensor& lse, std::int64_t ignore, bool need_hidden,
                               bool need_weight) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [gh, gw] =
        call_backward(gl, ge, labels, hidden, weight, lse, ignore, need_hidden, need_weight);
    return {gh, gw};
  }

  static variable_list backward(AutogradContext*, const variable_list&) {
    TORCH_CHECK(false,
                "cid_engine.lm_head_cross_entropy is differentiable once: its gradient has no "
                "gradient");
  }
};

// There is no forward-mode derivative.  A tensor with a tangent need not require a
// gradient, so this is looked at whether or not a graph is recorded: without the
// check the outputs would carry no tangent, which reads as a derivative of zero.
void refuse_tangents(const char* op, std::initializer_list<const at::Tensor*> tensors) {
  for (const auto* t : tensors)
    TORCH_CHECK(!t->defined() || !t->_fw_grad(/*level=*/0).defined(), "cid_engine.", op,
                " has no forward-mode derivative (dual tensors, torch.func.jvp)");
}

// Whether a graph is being recorded over any of the tensors; without one the
// nodes below would cost a call their set-up for nothing.
bool recording(std::initializer_list<const at::Tensor*> tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const auto* t : tensors)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

Pair forward_autograd(const at::Tensor& labels, const at::Tensor& hidden,
                      const at::Tensor& weight, std::int64_t ignore) {
  refuse_tangents("lm_head_cross_entropy", {&hidden, &weight});
  if (!recording({&hidden, &weight})) {
    at::AutoDispatchBelowADInplaceOrView below;
    return call_forward(labels, hidden, weight, ignore);
  }
  auto out = HeadLoss::apply(labels, hidden, weight, ignore);
  return {out[0], out[1]};
}

Pair backward_autograd(const std::optional<at::Tensor>& gl, const std::optional<at::Tensor>& ge,
                       const at::Tensor& labels, const at::Tensor& hidden,
                       const at::Tensor& weight, const at::Tensor& lse, std::int64_t ignore,
                       bool need_hidden, bool need_weight) {
  const at::Tensor none;
  const std::initializer_list<const at::Tensor*> inputs = {gl ? &*gl : &none, ge ? &*ge : &none,
                                                           &hidden, &weight, &lse};
  refuse_tangents("lm_head_cross_entropy_backward", inputs);
  if (!recording(inputs)) {
    at::AutoDispatchBelowADInplaceOrView below;
    return call_backward(gl, ge, labels, hidden, weight, lse, ignore, need_hidden, need_weight);
  }
  auto out = HeadLossBackward::apply(gl, ge, labels, hidden, weight, lse, ignore, need_hidden,
                                     need_weight);
  return {out[0], out[1]};
}

}  // namespace
}  // namespace cid::engine

TORCH_LIBRARY_IMPL(cid_engine, Autograd, m) {
  m.impl("lm_head_cross_entropy", TORCH_FN(cid::engine::forward_autograd));
  m.impl("lm_head_cross_entropy_backward", TORCH_FN(cid::engine::backward_autograd));
}
