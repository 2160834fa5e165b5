// The host path of the choice of experts (moe_ops.select_experts): argument checks, the node of the autograd graph and the launches.
#include "host_common.h"

#include <cmath>

namespace fp8gmm_host {
namespace {

// The chain from the weights of the chosen experts back to the scores.
struct SelectExpertsBackward : public Node {
  SavedVariable scores, selected;
  int64_t tokens = 0;
  fp8gmm_choice choice = {};
  at::ScalarType type = at::kBFloat16;

  std::string name() const override { return "SelectExpertsBackward"; }
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    scores.reset_data();
    selected.reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    const std::lock_guard<std::mutex> lock(mutex_);
    const bool graph = at::GradMode::is_enabled();
    variable_list result(1);
    const Tensor saved = scores.unpack();
    const Tensor grad = gradient_of_result(*this, grads);
    const c10::OptionalDeviceGuard guard(grad.device());
    {
      at::AutoGradMode no_grad(false);
      const Tensor s = saved.resolve_neg().contiguous(), chosen = selected.unpack().resolve_neg();
      TORCH_CHECK(s.scalar_type() == type && s.numel() == tokens * choice.experts && s.device() == grad.device() &&
                      chosen.scalar_type() == at::kLong && chosen.numel() == tokens * choice.top_k && chosen.is_contiguous() &&
                      chosen.device() == grad.device(),
                  "fp8_gmm_amd: a saved-tensor hook returned another tensor than was saved");
      const Tensor dw = grad.to(at::kFloat).contiguous();
      result[0] = at::empty(saved.sizes(), s.options());
      timed("select_experts_backward", 2 * s.numel() * (int64_t)s.element_size(), [&] {
        check(fp8gmm_select_experts_backward(ptr<void>(s), type_of(s, "scores"), tokens, &choice, ptr<int64_t>(chosen), ptr<float>(dw),
                                             ptr<void>(result[0]), current_stream(grad.device())));
      });
    }
    if (graph) refuse_second_derivative(result, "select_experts", {grad, saved});
    return result;
  }
};

std::pair<Tensor, Tensor> select_experts(const Tensor& scores, int64_t top_k, bool sigmoid, const std::optional<Tensor>& bias_,
                                         int64_t groups, int64_t top_groups, int64_t group_best, bool renormalize, double scale) {
  std::pair<Tensor, Tensor> out;
  with_python_errors([&] {
    py::gil_scoped_release no_gil;
    check_unwrapped("select_experts");
    check_plain(scores, "scores");
    type_of(scores, "scores");
    TORCH_CHECK(scores.dim() == 2, "fp8_gmm_amd: scores must be [tokens, experts], got ", scores.dim(), " dimensions");
    const int64_t tokens = scores.size(0), experts = scores.size(1);
    TORCH_CHECK(tokens <= INT32_MAX && experts >= 1 && experts <= FP8GMM_MAX_CHOICE_EXPERTS, "fp8_gmm_amd: between 1 and ",
                FP8GMM_MAX_CHOICE_EXPERTS, " experts are supported, got ", experts);
    TORCH_CHECK(groups >= 1 && groups <= FP8GMM_MAX_CHOICE_GROUPS && experts % groups == 0, "fp8_gmm_amd: ", experts,
                " experts cannot be cut into ", groups, " groups (at most ", FP8GMM_MAX_CHOICE_GROUPS, ", all of one size)");
    TORCH_CHECK(top_groups >= 1 && top_groups <= groups, "fp8_gmm_amd: top_groups must lie between 1 and ", groups, ", got ", top_groups);
    TORCH_CHECK(group_best == 1 || group_best == 2, "fp8_gmm_amd: group_best must be 1 or 2, got ", group_best);
    TORCH_CHECK(top_k >= 1 && top_k <= FP8GMM_MAX_CHOICES && top_k <= experts / groups * top_groups, "fp8_gmm_amd: top_k must lie between 1 and ",
                std::min<int64_t>(FP8GMM_MAX_CHOICES, experts / groups * top_groups), ", got ", top_k);
    TORCH_CHECK(std::isfinite((float)scale), "fp8_gmm_amd: scale must be a finite number");
    const Tensor bias = bias_.value_or(Tensor());
    if (bias.defined()) {
      check_plain(bias, "bias");
      TORCH_CHECK(bias.scalar_type() == at::kFloat && bias.dim() == 1 && bias.size(0) == experts && bias.device() == scores.device(),
                  "fp8_gmm_amd: bias must be float32 [experts] on the scores' device");
    }
    check_no_tangent({scores, bias}, "select_experts does");
    const c10::OptionalDeviceGuard guard(scores.device());
    const bool grad = at::GradMode::is_enabled() && wants_grad(scores);
    Tensor weights, selected;
    fp8gmm_choice choice = {};
    {
      at::AutoGradMode no_grad(false);
      const Tensor s = scores.contiguous(), b = bias.defined() ? bias.contiguous() : Tensor();
      weights = at::empty({tokens, top_k}, scores.options().dtype(at::kFloat));
      selected = at::empty({tokens, top_k}, scores.options().dtype(at::kLong));
      choice.bias = ptr<float>(b);
      choice.experts = (int)experts;
      choice.top_k = (int)top_k;
      choice.scoring = sigmoid ? FP8GMM_SCORING_SIGMOID : FP8GMM_SCORING_SOFTMAX;
      choice.groups = (int)groups;
      choice.top_groups = (int)top_groups;
      choice.group_best = (int)group_best;
      choice.renormalize = renormalize;
      choice.scale = (float)scale;
      timed("select_experts", s.numel() * (int64_t)s.element_size(), [&] {
        check(fp8gmm_select_experts(ptr<void>(s), type_of(s, "scores"), tokens, &choice, ptr<float>(weights), ptr<int64_t>(selected),
                                    current_stream(scores.device())));
      });
    }
    if (grad) {
      auto node = std::shared_ptr<SelectExpertsBackward>(new SelectExpertsBackward(), torch::autograd::deleteNode);
      node->set_next_edges(torch::autograd::collect_next_edges(scores));
      node->scores = SavedVariable(scores, false);
      node->selected = SavedVariable(selected, false);
      node->tokens = tokens;
      node->choice = choice;
      node->choice.bias = nullptr;   // a constant of the choice, and no part of the gradient
      node->type = scores.scalar_type();
      torch::autograd::set_history(weights, node);
    }
    out = {weights, selected};
    return Tensor();
  });
  return out;
}

}  // namespace

void define_routing(py::module_& m) { m.def("select_experts", &select_experts); }

}  // namespace fp8gmm_host
