// The host path of the optimizer's step over many tensors (backend.multi_adamw): argument checks and the table of the launches.
#include "host_common.h"

#include <ATen/MemoryOverlap.h>

#include <cmath>
#include <optional>
#include <variant>

namespace fp8gmm_host {
namespace {

typedef std::vector<Tensor> List;

// The tensors of anything that iterates over tensors (a step over 400 small ones 93 us, with pybind11's own conversion of lists 98).
List list_of(const py::object& from) {
  const py::object items = py::reinterpret_steal<py::object>(PySequence_Fast(from.ptr(), "fp8_gmm_amd: multi_adamw takes lists of tensors"));
  if (!items) throw py::error_already_set();
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(items.ptr());
  PyObject* const* const item = PySequence_Fast_ITEMS(items.ptr());
  List list;
  list.reserve(n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    if (!THPVariable_Check(item[i])) throw py::type_error("fp8_gmm_amd: multi_adamw takes lists of tensors");
    list.push_back(THPVariable_Unpack(item[i]));
  }
  return list;
}

// What a step writes: dense memory in the order of its parameter's elements.
void check_written(const Tensor& t, const Tensor& param, at::ScalarType type, const char* what) {
  check_plain(t, what);
  TORCH_CHECK(t.scalar_type() == type && t.sizes() == param.sizes() && t.device() == param.device(), "fp8_gmm_amd: ", what,
              " of multi_adamw must have its parameter's shape and device and be ", type, ", got ", t.scalar_type(), " ", t.sizes());
  TORCH_CHECK(pass_as_they_are(t, param), "fp8_gmm_amd: ", what,
              " of multi_adamw must be dense, its elements in the order of its parameter's");
}
void check_writable(const Tensor& t, const char* what) {
  TORCH_CHECK(!(at::GradMode::is_enabled() && t.requires_grad()), "fp8_gmm_amd: ", what,
              " of multi_adamw requires a gradient: step under torch.no_grad()");
  TORCH_CHECK(!t.is_inference() || c10::InferenceMode::is_enabled(), "fp8_gmm_amd: ", what,
              " of multi_adamw is an inference tensor, which is written in inference mode only");
}

// One number: of the host, or one that a replayed launch reads anew.  (A tensor comes first: it would pass for an integer.)
template <class T>
struct Number {
  T host;
  Tensor device;
};
template <class T>
Number<T> number(const std::variant<Tensor, T>& v, at::ScalarType type, const at::Device& device, const char* what) {
  if (const T* host = std::get_if<T>(&v)) return {*host, Tensor()};
  const Tensor& t = std::get<Tensor>(v);
  check_plain(t, what);
  TORCH_CHECK(t.scalar_type() == type && t.numel() == 1 && t.device() == device, "fp8_gmm_amd: ", what, " must be a number or one ", type,
              " on the parameters' device");
  return {T(), t};
}

void multi_adamw(const py::object& params_, const py::object& grads_, const py::object& exp_avgs_, const py::object& exp_avg_sqs_,
                 const std::variant<Tensor, int64_t>& step_, const std::variant<Tensor, double>& lr_, std::pair<double, double> betas,
                 double eps, double weight_decay, const std::optional<std::pair<py::object, py::object>>& scales_,
                 const std::optional<py::object>& masters_, const std::optional<Tensor>& norm, std::optional<double> max_norm) {
  const List params = list_of(params_), grads = list_of(grads_), exp_avgs = list_of(exp_avgs_), exp_avg_sqs = list_of(exp_avg_sqs_);
  std::optional<std::pair<List, List>> scales;
  if (scales_) scales.emplace(list_of(scales_->first), list_of(scales_->second));
  std::optional<List> masters;
  if (masters_) masters.emplace(list_of(*masters_));
  py::gil_scoped_release no_gil;
  check_unwrapped("multi_adamw");
  const size_t n = params.size();
  TORCH_CHECK(n > 0, "fp8_gmm_amd: multi_adamw needs at least one tensor");
  TORCH_CHECK(grads.size() == n && exp_avgs.size() == n && exp_avg_sqs.size() == n && (!masters || masters->size() == n) &&
                  (!scales || (scales->first.size() == n && scales->second.size() == n)),
              "fp8_gmm_amd: multi_adamw needs a gradient, both moments and, where given, both scales and a master for every parameter");
  TORCH_CHECK(norm.has_value() == max_norm.has_value(), "fp8_gmm_amd: norm and max_norm go together");
  check_plain(params[0], "a parameter");
  const at::Device device = params[0].device();
  const Number<int64_t> step = number<int64_t>(step_, at::kLong, device, "step");
  const Number<double> lr = number<double>(lr_, at::kFloat, device, "lr");
  TORCH_CHECK(step.device.defined() || step.host >= 1, "fp8_gmm_amd: step counts from 1, got ", step.host);
  TORCH_CHECK(lr.device.defined() || (lr.host >= 0 && std::isfinite(lr.host)), "fp8_gmm_amd: lr must be a number, not negative");
  TORCH_CHECK(betas.first >= 0 && betas.first < 1 && betas.second >= 0 && betas.second < 1, "fp8_gmm_amd: betas must lie in [0, 1)");
  TORCH_CHECK(eps >= 0 && std::isfinite(eps) && weight_decay >= 0 && std::isfinite(weight_decay),
              "fp8_gmm_amd: eps and weight_decay must be numbers, not negative");
  if (norm.has_value()) {
    check_plain(*norm, "norm");
    TORCH_CHECK(norm->scalar_type() == at::kFloat && norm->numel() == 1 && norm->device() == device,
                "fp8_gmm_amd: norm must be one float32 on the parameters' device");
    TORCH_CHECK(*max_norm >= 0, "fp8_gmm_amd: max_norm must be a number, not negative");
  }
  for (const List* list : {&params, &grads, &exp_avgs, &exp_avg_sqs}) check_no_tangent(*list, "multi_adamw does");
  if (masters) check_no_tangent(*masters, "multi_adamw does");
  for (const Tensor* t : {&step.device, &lr.device})
    if (t->defined()) check_no_tangent({*t}, "multi_adamw does");
  if (norm.has_value()) check_no_tangent({*norm}, "multi_adamw does");

  const at::ScalarType moment = scales ? at::kFloat8_e4m3fn : at::kFloat;
  int64_t bytes = 0;
  for (size_t i = 0; i < n; ++i) {
    const Tensor &p = params[i], &g = grads[i];
    check_plain(p, "a parameter");
    type_of(p, "a parameter");
    TORCH_CHECK(p.device() == device, "fp8_gmm_amd: all tensors of one call must live on the same device");
    TORCH_CHECK(dense(p), "fp8_gmm_amd: a parameter of multi_adamw must be dense");
    TORCH_CHECK(p.numel() <= (int64_t)1 << 32, "fp8_gmm_amd: a parameter of multi_adamw has at most 2^32 elements");
    check_writable(p, "a parameter");
    TORCH_CHECK(g.is_cuda() && g.layout() == at::kStrided, "fp8_gmm_amd: a gradient of multi_adamw must be a dense GPU tensor");
    TORCH_CHECK(g.sizes() == p.sizes() && g.device() == device && (g.scalar_type() == p.scalar_type() || g.scalar_type() == at::kFloat),
                "fp8_gmm_amd: a gradient of multi_adamw must have its parameter's shape and device, and its type or float32");
    check_written(exp_avgs[i], p, moment, "exp_avg");
    check_written(exp_avg_sqs[i], p, moment, "exp_avg_sq");
    check_writable(exp_avgs[i], "exp_avg");
    check_writable(exp_avg_sqs[i], "exp_avg_sq");
    if (masters) {
      TORCH_CHECK(p.scalar_type() != at::kFloat, "fp8_gmm_amd: a float32 parameter is its own master");
      check_written((*masters)[i], p, at::kFloat, "a master");
      check_writable((*masters)[i], "a master");
    }
    if (scales) {
      const int64_t blocks = (p.numel() + FP8GMM_ADAMW_BLOCK - 1) / FP8GMM_ADAMW_BLOCK;
      for (const Tensor* t : {&scales->first[i], &scales->second[i]}) {
        check_plain(*t, "scales");
        TORCH_CHECK(t->scalar_type() == at::kFloat && t->dim() == 1 && t->size(0) == blocks && t->is_contiguous() && t->device() == device,
                    "fp8_gmm_amd: scales of multi_adamw must be contiguous float32 [", blocks, "], one for ", FP8GMM_ADAMW_BLOCK, " elements");
        check_writable(*t, "scales");
      }
    }
    bytes += p.numel() * (2 * (int64_t)p.element_size() + (int64_t)g.element_size() + 4 * (int64_t)exp_avgs[i].element_size());
    if (masters) bytes += p.numel() * (8 - (int64_t)p.element_size());
  }

  at::AutoGradMode no_grad(false);
  const c10::OptionalDeviceGuard guard(device);
  std::vector<fp8gmm_adamw_tensor> list(n);
  List kept;   // gradients in the order of their parameters' elements
  kept.reserve(n);
  for (size_t i = 0; i < n; ++i) {
    const Tensor& p = params[i];
    const Tensor* grad = &grads[i];
    if (grad->is_neg() || !pass_as_they_are(*grad, p)) {
      kept.push_back(at::empty_strided(p.sizes(), p.strides(), grad->options()).copy_(*grad));
      grad = &kept.back();
    }
    const Tensor& g = *grad;
    list[i] = {ptr<void>(p),
               ptr<void>(g),
               ptr<void>(exp_avgs[i]),
               ptr<void>(exp_avg_sqs[i]),
               scales ? ptr<float>(scales->first[i]) : nullptr,
               scales ? ptr<float>(scales->second[i]) : nullptr,
               masters ? ptr<float>((*masters)[i]) : nullptr,
               p.numel(),
               type_of(p, ""),
               type_of(g, "")};
  }
  fp8gmm_adamw_step a = {};
  a.lr = lr.host;
  a.beta1 = betas.first;
  a.beta2 = betas.second;
  a.eps = eps;
  a.weight_decay = weight_decay;
  a.max_norm = max_norm.value_or(0.);
  a.norm = norm.has_value() ? ptr<float>(*norm) : nullptr;
  a.step_dev = ptr<int64_t>(step.device);
  a.lr_dev = ptr<float>(lr.device);
  a.step = step.host;
  a.bits = scales ? 8 : 32;
  timed("multi_adamw", bytes, [&] {
    const int rc = fp8gmm_multi_adamw(list.data(), (int)n, &a, current_stream(device));
    TORCH_CHECK(rc != FP8GMM_ERR_BAD_ARGUMENT, "fp8_gmm_amd: what multi_adamw writes overlaps another tensor of the call");
    check(rc);
  });
  const auto written = [](const List& tensors) {
    for (const Tensor& t : tensors) torch::autograd::impl::bump_version(t);
  };
  written(params);
  written(exp_avgs);
  written(exp_avg_sqs);
  if (masters) written(*masters);
  if (scales) {
    written(scales->first);
    written(scales->second);
  }
}

}  // namespace

void define_adamw(py::module_& m) { m.def("multi_adamw", &multi_adamw); }

}  // namespace fp8gmm_host
