// The host path of the operators around the routed layers: the norms of rows and embedding with their gradients (layers.py), the
// norm of many tensors and their scaling by it (backend.multi_norm, multi_clip).  A short call is bound by its host, so the argument
// checks, the nodes of the autograd graph and the launches' tables are native as in host_passes.cpp.
#include "host_common.h"

#include <ATen/MemoryOverlap.h>

#include <algorithm>
#include <cmath>
#include <limits>

namespace fp8gmm_host {
namespace {

// ---- layer norm ------------------------------------------------------------------------------------------------------
// The rows of a tensor of any shape, and their pitch: as they are where the columns are neighbours, otherwise copied.
struct Rows {
  Tensor t;
  int64_t pitch;
};
Rows rows_of(const Tensor& t, int64_t rows, int64_t cols) {
  if (t.is_contiguous()) return {t, cols};
  Tensor flat = t.reshape({rows, cols});
  if ((cols > 1 && flat.stride(1) != 1) || (rows > 1 && flat.stride(0) < cols)) flat = flat.contiguous();
  return {flat, rows > 1 ? flat.stride(0) : cols};
}

struct LayerNormBackward : public Node {
  SavedVariable x, weight;
  Tensor stats;   // mean and rstd of every row
  int64_t rows = 0, cols = 0;
  int type = 0, param_type = 0;
  bool bias = false;

  std::string name() const override { return "LayerNormBackward"; }
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    x.reset_data();
    weight.reset_data();
    stats.reset();
  }
  variable_list apply(variable_list&& grads) override {
    const std::lock_guard<std::mutex> lock(mutex_);
    const bool graph = at::GradMode::is_enabled();
    variable_list result(bias ? 3 : 2);
    const Tensor xs = x.unpack(), w = weight.unpack();
    const Tensor grad = gradient_of_result(*this, grads);
    const c10::OptionalDeviceGuard guard(grad.device());
    {
      at::AutoGradMode no_grad(false);
      TORCH_CHECK(xs.device() == grad.device() && xs.numel() == rows * cols && xs.scalar_type() == grad.scalar_type() &&
                      w.device() == grad.device() && w.numel() == cols && w.is_contiguous() && type_of(w, "weight") == param_type &&
                      type_of(xs, "input") == type,
                  "fp8_gmm_amd: a saved-tensor hook returned another tensor than was saved");
      const Rows from = rows_of(xs.resolve_neg(), rows, cols), dy = rows_of(grad, rows, cols);
      const Tensor params = w.resolve_neg();
      if (task_should_compute_output(0)) result[0] = at::empty(xs.sizes(), xs.options());
      if (task_should_compute_output(1)) result[1] = at::empty({cols}, w.options());
      if (bias && task_should_compute_output(2)) result[2] = at::empty({cols}, w.options());
      Tensor work;
      size_t bytes = 0;
      if (rows > 0 && (result[1].defined() || (bias && result[2].defined()))) {
        bytes = fp8gmm_layer_norm_workspace_bytes(rows, (int)cols, type);
        work = at::empty({(int64_t)bytes}, xs.options().dtype(at::kByte));
      }
      timed("layer_norm_backward", (2 + result[0].defined()) * xs.numel() * (int64_t)xs.element_size(), [&] {
        check(fp8gmm_layer_norm_backward(ptr<void>(dy.t), dy.pitch, ptr<void>(from.t), from.pitch, ptr<void>(params), ptr<float>(stats),
                                         ptr<float>(stats) + rows, ptr<void>(result[0]), ptr<void>(result[1]),
                                         bias ? ptr<void>(result[2]) : nullptr, rows, (int)cols, type, param_type, ptr<void>(work),
                                         bytes, current_stream(grad.device())));
      });
    }
    if (graph) refuse_second_derivative(result, "layer_norm", {grad, xs, w});
    return result;
  }
};

Tensor layer_norm(const Tensor& x, const Tensor& weight, const std::optional<Tensor>& bias_, double eps) {
  return with_python_errors([&] {
    py::gil_scoped_release no_gil;
    check_unwrapped("layer_norm");
    const Tensor bias = bias_.value_or(Tensor());
    check_plain(x, "the input of layer_norm");
    check_plain(weight, "weight");
    const int type = type_of(x, "the input of layer_norm"), param_type = type_of(weight, "weight");
    TORCH_CHECK(param_type == type || param_type == FP8GMM_TYPE_FP32, "fp8_gmm_amd: weight must have the input's type or be float32");
    TORCH_CHECK(x.dim() >= 1 && weight.dim() == 1 && x.size(-1) == weight.size(0) && weight.size(0) >= 1,
                "fp8_gmm_amd: weight must be 1-D with as many elements as the input has columns, at least one");
    TORCH_CHECK(weight.device() == x.device(), "fp8_gmm_amd: all tensors of one call must live on the same device");
    if (bias.defined()) {
      check_plain(bias, "bias");
      TORCH_CHECK(bias.sizes() == weight.sizes() && bias.scalar_type() == weight.scalar_type() && bias.device() == x.device(),
                  "fp8_gmm_amd: bias must have the weight's shape, type and device");
    }
    TORCH_CHECK(eps >= 0 && std::isfinite(eps), "fp8_gmm_amd: eps must be a number, not negative");
    check_no_tangent({x, weight, bias}, "layer_norm does");
    const int64_t cols = x.size(-1), rows = x.numel() / cols;
    TORCH_CHECK(cols <= 1 << 30 && rows <= INT32_MAX, "fp8_gmm_amd: at most 2^30 columns and 2^31 - 1 rows are supported");
    const c10::OptionalDeviceGuard guard(x.device());
    const bool grad = at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(weight) || wants_grad(bias));
    Tensor y, stats, w;
    {
      at::AutoGradMode no_grad(false);
      const Rows from = rows_of(x, rows, cols);
      w = weight.contiguous();
      const Tensor b = bias.defined() ? bias.contiguous() : Tensor();
      y = at::empty(x.sizes(), x.options());
      if (grad) stats = at::empty({2, rows}, x.options().dtype(at::kFloat));
      float* const mean = ptr<float>(stats);
      timed("layer_norm", 2 * x.numel() * (int64_t)x.element_size(), [&] {
        check(fp8gmm_layer_norm(ptr<void>(from.t), from.pitch, ptr<void>(w), ptr<void>(b), ptr<void>(y), mean,
                                mean != nullptr ? mean + rows : nullptr, rows, (int)cols, (float)eps, type, param_type, current_stream(x.device())));
      });
    }
    if (grad) {
      auto node = std::shared_ptr<LayerNormBackward>(new LayerNormBackward(), torch::autograd::deleteNode);
      node->bias = bias.defined();
      if (bias.defined()) node->set_next_edges(torch::autograd::collect_next_edges(x, weight, bias));
      else node->set_next_edges(torch::autograd::collect_next_edges(x, weight));
      node->x = SavedVariable(x, false);
      node->weight = SavedVariable(weight.is_contiguous() ? weight : w, false);
      node->stats = stats;
      node->rows = rows;
      node->cols = cols;
      node->type = type;
      node->param_type = param_type;
      torch::autograd::set_history(y, node);
    }
    return y;
  });
}

// ---- root-mean-square norm -------------------------------------------------------------------------------------------
struct RmsNormBackward : public Node {
  SavedVariable h, weight;
  Tensor rstd;
  int64_t rows = 0, cols = 0;
  int type = 0, param_type = 0;
  bool residual = false;

  std::string name() const override { return "RmsNormBackward"; }
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    h.reset_data();
    weight.reset_data();
    rstd.reset();
  }
  variable_list apply(variable_list&& grads) override {
    const std::lock_guard<std::mutex> lock(mutex_);
    const bool graph = at::GradMode::is_enabled();
    variable_list result(residual ? 3 : 2);
    // with a residual h is a result of this node
    const Tensor hs = residual ? h.unpack(shared_from_this()) : h.unpack(), w = weight.unpack();
    const Tensor grad = grads[0].defined() || !(residual && grads[1].defined()) ? gradient_of_result(*this, grads) : Tensor();
    const Tensor grad_h = residual && grads[1].defined() ? plain_gradient(grads[1]) : Tensor();
    const bool want_x = task_should_compute_output(0) || (residual && task_should_compute_output(2));
    if (!grad.defined()) {   // the sum alone was used
      if (task_should_compute_output(0)) result[0] = grads[1];
      if (task_should_compute_output(2)) result[2] = grads[1];
      return result;
    }
    const c10::OptionalDeviceGuard guard(grad.device());
    Tensor dx;
    {
      at::AutoGradMode no_grad(false);
      TORCH_CHECK(hs.device() == grad.device() && hs.numel() == rows * cols && hs.scalar_type() == grad.scalar_type() &&
                      w.device() == grad.device() && w.numel() == cols && w.is_contiguous() && type_of(w, "weight") == param_type &&
                      type_of(hs, "input") == type,
                  "fp8_gmm_amd: a saved-tensor hook returned another tensor than was saved");
      const Rows from = rows_of(hs.resolve_neg(), rows, cols), dy = rows_of(grad, rows, cols);
      const Rows dh = grad_h.defined() ? rows_of(grad_h, rows, cols) : Rows{Tensor(), cols};
      const Tensor params = w.resolve_neg();
      if (want_x) dx = at::empty(hs.sizes(), hs.options());
      if (task_should_compute_output(1)) result[1] = at::empty({cols}, w.options());
      Tensor work;
      size_t bytes = 0;
      if (rows > 0 && result[1].defined()) {
        bytes = fp8gmm_rms_norm_workspace_bytes(rows, (int)cols, type);
        work = at::empty({(int64_t)bytes}, hs.options().dtype(at::kByte));
      }
      timed("rms_norm_backward", (2 + dx.defined() + grad_h.defined()) * hs.numel() * (int64_t)hs.element_size(), [&] {
        check(fp8gmm_rms_norm_backward(ptr<void>(dy.t), dy.pitch, ptr<void>(dh.t), dh.pitch, ptr<void>(from.t), from.pitch,
                                       ptr<void>(params), ptr<float>(rstd), ptr<void>(dx), ptr<void>(result[1]), rows, (int)cols, type,
                                       param_type, ptr<void>(work), bytes, current_stream(grad.device())));
      });
    }
    if (task_should_compute_output(0)) result[0] = dx;
    if (residual && task_should_compute_output(2)) result[2] = dx;
    if (graph) {
      variable_list from = {grad, hs, w};
      if (grad_h.defined()) from.push_back(grad_h);
      refuse_second_derivative(result, "rms_norm", from);
    }
    return result;
  }
};

// What both root-mean-square norms ask of their rows
struct RmsRows {
  int type, param_type;
  int64_t rows, cols;
};
RmsRows check_rms(const Tensor& x, const Tensor& weight, const Tensor& residual, double eps, const char* name, const char* does) {
  check_unwrapped(name);
  check_plain(x, "the input of a norm");
  check_plain(weight, "weight");
  const int type = type_of(x, "the input of a norm"), param_type = type_of(weight, "weight");
  TORCH_CHECK(param_type == type || param_type == FP8GMM_TYPE_FP32, "fp8_gmm_amd: weight must have the input's type or be float32");
  TORCH_CHECK(x.dim() >= 1 && weight.dim() == 1 && x.size(-1) == weight.size(0) && weight.size(0) >= 1,
              "fp8_gmm_amd: weight must be 1-D with as many elements as the input has columns, at least one");
  TORCH_CHECK(weight.device() == x.device(), "fp8_gmm_amd: all tensors of one call must live on the same device");
  if (residual.defined()) {
    check_plain(residual, "residual");
    TORCH_CHECK(residual.sizes() == x.sizes() && residual.scalar_type() == x.scalar_type() && residual.device() == x.device(),
                "fp8_gmm_amd: residual must have the input's shape, type and device");
  }
  TORCH_CHECK(eps >= 0 && std::isfinite(eps), "fp8_gmm_amd: eps must be a number, not negative");
  check_no_tangent({x, weight, residual}, does);
  const int64_t cols = x.size(-1), rows = x.numel() / cols;
  TORCH_CHECK(cols <= 1 << 30 && rows <= INT32_MAX, "fp8_gmm_amd: at most 2^30 columns and 2^31 - 1 rows are supported");
  return {type, param_type, rows, cols};
}

// (y, h): h the rows that are normed, undefined without a residual
std::pair<Tensor, Tensor> rms_norm(const Tensor& x, const Tensor& weight, double eps, const std::optional<Tensor>& residual_) {
  std::pair<Tensor, Tensor> out;
  with_python_errors([&] {
    py::gil_scoped_release no_gil;
    const Tensor residual = residual_.value_or(Tensor());
    const RmsRows r = check_rms(x, weight, residual, eps, "rms_norm", "rms_norm does");
    const c10::OptionalDeviceGuard guard(x.device());
    const bool grad = at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(weight) || wants_grad(residual));
    Tensor y, h, rstd, w;
    {
      at::AutoGradMode no_grad(false);
      const Rows from = rows_of(x, r.rows, r.cols), add = residual.defined() ? rows_of(residual, r.rows, r.cols) : Rows{Tensor(), r.cols};
      w = weight.contiguous();
      y = at::empty(x.sizes(), x.options());
      if (residual.defined()) h = at::empty(x.sizes(), x.options());
      if (grad) rstd = at::empty({r.rows}, x.options().dtype(at::kFloat));
      timed("rms_norm", (residual.defined() ? 4 : 2) * x.numel() * (int64_t)x.element_size(), [&] {
        check(fp8gmm_rms_norm(ptr<void>(from.t), from.pitch, ptr<void>(add.t), add.pitch, ptr<void>(w), ptr<void>(y), ptr<void>(h),
                              ptr<float>(rstd), r.rows, (int)r.cols, (float)eps, r.type, r.param_type, current_stream(x.device())));
      });
    }
    if (grad) {
      auto node = std::shared_ptr<RmsNormBackward>(new RmsNormBackward(), torch::autograd::deleteNode);
      if (residual.defined()) node->set_next_edges(torch::autograd::collect_next_edges(x, weight, residual));
      else node->set_next_edges(torch::autograd::collect_next_edges(x, weight));
      node->rstd = rstd;
      node->rows = r.rows;
      node->cols = r.cols;
      node->type = r.type;
      node->param_type = r.param_type;
      node->residual = residual.defined();
      torch::autograd::set_history(y, node);
      if (residual.defined()) torch::autograd::set_history(h, node);
      node->h = residual.defined() ? SavedVariable(h, true) : SavedVariable(x, false);
      node->weight = SavedVariable(weight.is_contiguous() ? weight : w, false);
    }
    out = {y, h};
    return Tensor();
  });
  return out;
}

// (q, scale_inv of the rows or undefined, h or undefined)
std::tuple<Tensor, Tensor, Tensor> rms_norm_fp8(const Tensor& x, const Tensor& weight, double eps, const std::optional<Tensor>& residual_,
                                                const std::optional<Tensor>& scale_, const std::optional<Tensor>& amax_,
                                                at::ScalarType format) {
  py::gil_scoped_release no_gil;
  const Tensor residual = residual_.value_or(Tensor()), scale = scale_.value_or(Tensor()), amax = amax_.value_or(Tensor());
  const RmsRows r = check_rms(x, weight, residual, eps, "rms_norm_fp8", "rms_norm_fp8 does");
  TORCH_CHECK(format == at::kFloat8_e4m3fn || format == at::kFloat8_e5m2,
              "fp8_gmm_amd: dtype must be torch.float8_e4m3fn or torch.float8_e5m2");
  TORCH_CHECK(!(at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(weight) || wants_grad(residual))),
              "fp8_gmm_amd: rms_norm_fp8 takes no gradients: call it under torch.no_grad() or on detached tensors");
  for (const Tensor& t : {scale, amax}) {
    if (!t.defined()) continue;
    check_plain(t, "scale and amax");
    TORCH_CHECK(t.scalar_type() == at::kFloat && t.numel() == 1 && t.device() == x.device(),
                "fp8_gmm_amd: scale and amax must be one float32 each, on the input's device");
  }
  TORCH_CHECK(scale.defined() || !amax.defined(), "fp8_gmm_amd: amax is recorded with a scale of the tensor");
  if (amax.defined()) {
    TORCH_CHECK(!amax.is_inference() || c10::InferenceMode::is_enabled(),
                "fp8_gmm_amd: amax is an inference tensor, which is written in inference mode only");
    TORCH_CHECK(!(at::GradMode::is_enabled() && amax.requires_grad()), "fp8_gmm_amd: amax requires a gradient");
    TORCH_CHECK(scale.data_ptr() != amax.data_ptr(), "fp8_gmm_amd: scale and amax must not share memory");
  }
  at::AutoGradMode no_grad(false);
  const c10::OptionalDeviceGuard guard(x.device());
  const Rows from = rows_of(x, r.rows, r.cols), add = residual.defined() ? rows_of(residual, r.rows, r.cols) : Rows{Tensor(), r.cols};
  const Tensor w = weight.contiguous();
  const Tensor q = at::empty(x.sizes(), x.options().dtype(format));
  Tensor h, scale_inv;
  if (residual.defined()) h = at::empty(x.sizes(), x.options());
  if (!scale.defined()) scale_inv = at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
  timed("rms_norm_fp8", x.numel() * ((residual.defined() ? 3 : 1) * (int64_t)x.element_size() + 1), [&] {
    check(fp8gmm_rms_norm_fp8(ptr<void>(from.t), from.pitch, ptr<void>(add.t), add.pitch, ptr<void>(w), ptr<void>(q), ptr<void>(h),
                              ptr<float>(scale), ptr<float>(amax), ptr<float>(scale_inv), r.rows, (int)r.cols, (float)eps, r.type,
                              r.param_type, format == at::kFloat8_e4m3fn ? FP8GMM_E4M3 : FP8GMM_E5M2, current_stream(x.device())));
  });
  if (amax.defined()) torch::autograd::impl::bump_version(amax);
  return {q, scale_inv, h};
}

// ---- embedding -------------------------------------------------------------------------------------------------------
struct EmbeddingBackward : public Node {
  SavedVariable ids;
  int64_t tokens = 0, table = 0, cols = 0, padding = -1;
  at::ScalarType id_type = at::kLong;
  double scale = 1;

  std::string name() const override { return "EmbeddingBackward"; }
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    ids.reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    const std::lock_guard<std::mutex> lock(mutex_);
    const bool graph = at::GradMode::is_enabled();
    const Tensor list = ids.unpack().resolve_neg();
    variable_list result(1);
    const Tensor grad = gradient_of_result(*this, grads);
    const c10::OptionalDeviceGuard guard(grad.device());
    {
      at::AutoGradMode no_grad(false);
      TORCH_CHECK(list.device() == grad.device() && list.numel() == tokens && list.scalar_type() == id_type && list.is_contiguous(),
                  "fp8_gmm_amd: a saved-tensor hook returned another tensor than was saved");
      const Tensor dy = grad.contiguous();
      const int type = type_of(dy, "gradient");
      result[0] = at::empty({table, cols}, dy.options());
      const size_t bytes = fp8gmm_embedding_workspace_bytes(tokens, table, (int)cols, type);
      Tensor work;   // short batches need none
      if (bytes > 0) work = at::empty({(int64_t)bytes}, dy.options().dtype(at::kByte));
      timed("embedding_backward", (dy.numel() + result[0].numel()) * (int64_t)dy.element_size(), [&] {
        check(fp8gmm_embedding_backward(ptr<void>(list), id_type == at::kLong, tokens, ptr<void>(dy), ptr<void>(result[0]), table,
                                        (int)cols, (float)scale, padding, type, ptr<void>(work), bytes, current_stream(grad.device())));
      });
    }
    if (graph) refuse_second_derivative(result, "embedding", {grad});
    return result;
  }
};

Tensor embedding(const Tensor& ids_, const Tensor& weight, double scale, std::optional<int64_t> padding_idx) {
  return with_python_errors([&] {
    py::gil_scoped_release no_gil;
    check_unwrapped("embedding");
    check_plain(ids_, "ids");
    check_plain(weight, "weight");
    TORCH_CHECK(ids_.scalar_type() == at::kLong || ids_.scalar_type() == at::kInt, "fp8_gmm_amd: ids must be int64 or int32, got ",
                ids_.scalar_type());
    const int type = type_of(weight, "weight");
    TORCH_CHECK(weight.dim() == 2 && weight.is_contiguous(), "fp8_gmm_amd: weight must be a contiguous table [rows, columns]");
    TORCH_CHECK(weight.device() == ids_.device(), "fp8_gmm_amd: all tensors of one call must live on the same device");
    TORCH_CHECK(std::isfinite((float)scale), "fp8_gmm_amd: scale must be a finite number");
    const int64_t table = weight.size(0), cols = weight.size(1), tokens = ids_.numel();
    TORCH_CHECK(cols <= 1 << 23 && table < INT32_MAX && tokens <= 1 << 28,
                "fp8_gmm_amd: at most 2^23 columns, 2^31 - 2 rows and 2^28 ids are supported");
    int64_t padding = -1;
    if (padding_idx.has_value()) {
      TORCH_CHECK(*padding_idx >= -table && *padding_idx < table, "fp8_gmm_amd: padding_idx must be a row of the table");
      padding = *padding_idx < 0 ? *padding_idx + table : *padding_idx;
    }
    check_no_tangent({weight}, "embedding does");
    const c10::OptionalDeviceGuard guard(weight.device());
    const Tensor ids = ids_.contiguous();
    std::vector<int64_t> sizes = ids.sizes().vec();
    sizes.push_back(cols);
    const bool grad = at::GradMode::is_enabled() && wants_grad(weight);
    Tensor y;
    {
      at::AutoGradMode no_grad(false);
      y = at::empty(sizes, weight.options());
      timed("embedding", 2 * y.numel() * (int64_t)y.element_size(), [&] {
        check(fp8gmm_embedding(ptr<void>(ids), ids.scalar_type() == at::kLong, tokens, ptr<void>(weight), table, (int)cols,
                               (float)scale, type, ptr<void>(y), current_stream(weight.device())));
      });
    }
    if (grad) {
      auto node = std::shared_ptr<EmbeddingBackward>(new EmbeddingBackward(), torch::autograd::deleteNode);
      node->set_next_edges(torch::autograd::collect_next_edges(weight));
      node->ids = SavedVariable(ids, false);
      node->tokens = tokens;
      node->table = table;
      node->cols = cols;
      node->padding = padding;
      node->id_type = ids.scalar_type();
      node->scale = scale;
      torch::autograd::set_history(y, node);
    }
    return y;
  });
}

// ---- norm of many tensors --------------------------------------------------------------------------------------------
void check_list(const std::vector<Tensor>& tensors, const char* what) {
  TORCH_CHECK(!tensors.empty(), "fp8_gmm_amd: ", what, " needs at least one tensor");
  for (const Tensor& t : tensors) {
    check_plain(t, what);
    type_of(t, what);
    TORCH_CHECK(t.device() == tensors[0].device(), "fp8_gmm_amd: all tensors of one call must live on the same device");
  }
}

int64_t bytes_of(const std::vector<Tensor>& tensors) {
  int64_t bytes = 0;
  for (const Tensor& t : tensors) bytes += t.numel() * (int64_t)t.element_size();
  return bytes;
}

Tensor multi_norm(const std::vector<Tensor>& tensors) {
  py::gil_scoped_release no_gil;
  check_unwrapped("multi_norm");
  check_list(tensors, "multi_norm");
  check_no_tangent(tensors, "multi_norm does");
  at::AutoGradMode no_grad(false);
  const at::Device device = tensors[0].device();
  const c10::OptionalDeviceGuard guard(device);
  std::vector<fp8gmm_norm_tensor> list(tensors.size());
  std::vector<Tensor> kept;
  for (size_t i = 0; i < tensors.size(); ++i) {
    Tensor t = tensors[i];
    if (!dense(t)) kept.push_back(t = t.contiguous());
    list[i] = {ptr<void>(t), nullptr, t.numel(), type_of(t, ""), 0};
  }
  const auto options = at::TensorOptions().device(device);
  const Tensor norm = at::empty({}, options.dtype(at::kFloat));
  const size_t bytes = fp8gmm_multi_norm_workspace_bytes((int)list.size());
  const Tensor work = at::empty({(int64_t)bytes}, options.dtype(at::kByte));
  timed("multi_norm", bytes_of(tensors), [&] {
    check(fp8gmm_multi_norm(list.data(), (int)list.size(), ptr<float>(norm), ptr<void>(work), bytes, current_stream(device)));
  });
  return norm;
}

// Where a tensor lies, in bytes: from its first element to behind its last one, and the rows in that where it consists of rows of
// one pitch (0: of none, or of one).
struct Place {
  uintptr_t begin, end;
  uintptr_t width, pitch;
};
Place place_of(const Tensor& t) {
  int64_t last = 0, width = 1, pitch = 0, span = 0;
  bool rows = true;
  for (int64_t d = t.dim() - 1; d >= 0; --d) {
    const int64_t size = t.size(d), stride = t.stride(d);
    if (size == 1) continue;
    last += (size - 1) * stride;
    if (pitch == 0 && stride == width) width *= size;
    else if (pitch == 0 || stride == span) span = stride * size, pitch = pitch == 0 ? stride : pitch;
    else rows = false;
  }
  const uintptr_t begin = reinterpret_cast<uintptr_t>(t.data_ptr()), size = t.element_size();
  return {begin, begin + (uintptr_t)(last + 1) * size, (uintptr_t)width * size, rows ? (uintptr_t)pitch * size : 0};
}
// Whether they lie apart: by their ends, or as slices of the columns of one buffer.  What cannot be told apart so counts as shared.
bool apart(const Place& a, const Place& b) {
  if (a.end <= b.begin || b.end <= a.begin) return true;
  if (a.begin > b.begin) return apart(b, a);
  const uintptr_t from = a.pitch != 0 && a.pitch == b.pitch ? (b.begin - a.begin) % a.pitch : 0;
  return from >= a.width && from + b.width <= a.pitch;
}

// A copy stands in for a tensor or its result where their elements do not pass as they are, so the library does not see where
// those lie.
void check_copied(const std::vector<Tensor>& tensors, const std::vector<Tensor>& outs) {
  for (size_t i = 0; i < outs.size(); ++i) {
    const Tensor &in = tensors[i], &out = outs[i];
    if (out.numel() == 0 || pass_as_they_are(in, out)) continue;
    const Place read = place_of(in), written = place_of(out);
    const bool in_place = in.data_ptr() == out.data_ptr() && in.scalar_type() == out.scalar_type() && same_order(in, out);
    bool shared = !in_place && !apart(read, written);
    for (size_t j = 0; j < outs.size(); ++j) {
      if (j == i || outs[j].numel() == 0) continue;
      const Place other = place_of(outs[j]);
      shared = shared || !apart(written, other) || !apart(read, other) || !apart(written, place_of(tensors[j]));
    }
    TORCH_CHECK(!shared, "fp8_gmm_amd: a result of multi_clip overlaps another tensor of the call");
  }
}

Tensor multi_clip(const std::vector<Tensor>& tensors, const std::vector<Tensor>& outs, double max_norm) {
  py::gil_scoped_release no_gil;
  check_unwrapped("multi_clip");
  check_list(tensors, "multi_clip");
  TORCH_CHECK(outs.size() == tensors.size(), "fp8_gmm_amd: multi_clip needs a result for every tensor");
  check_list(outs, "multi_clip");
  check_no_tangent(tensors, "multi_clip does");
  check_no_tangent(outs, "multi_clip does");
  TORCH_CHECK(outs[0].device() == tensors[0].device(), "fp8_gmm_amd: all tensors of one call must live on the same device");
  TORCH_CHECK(max_norm >= 0, "fp8_gmm_amd: max_norm must be a number, not negative");
  for (size_t i = 0; i < tensors.size(); ++i) {
    TORCH_CHECK(outs[i].sizes() == tensors[i].sizes() &&
                    (outs[i].scalar_type() == tensors[i].scalar_type() || outs[i].scalar_type() == at::kFloat),
                "fp8_gmm_amd: results of multi_clip have their tensors' shapes, and their types or float32");
    TORCH_CHECK(!(at::GradMode::is_enabled() && outs[i].requires_grad()), "fp8_gmm_amd: a result of multi_clip requires a gradient");
    TORCH_CHECK(!outs[i].is_inference() || c10::InferenceMode::is_enabled(),
                "fp8_gmm_amd: a result of multi_clip is an inference tensor, which is written in inference mode only");
    at::assert_no_internal_overlap(outs[i]);
  }
  check_copied(tensors, outs);
  at::AutoGradMode no_grad(false);
  const at::Device device = tensors[0].device();
  const c10::OptionalDeviceGuard guard(device);
  std::vector<fp8gmm_norm_tensor> list(tensors.size());
  std::vector<Tensor> kept;
  std::vector<std::pair<Tensor, Tensor>> copies;   // results that are copied to where they belong
  for (size_t i = 0; i < tensors.size(); ++i) {
    Tensor in = tensors[i], out = outs[i];
    if (!pass_as_they_are(in, out)) {   // element by element, in one order
      in = in.contiguous();
      kept.push_back(in);
      if (!out.is_contiguous()) {
        out = at::empty(out.sizes(), out.options());
        copies.emplace_back(outs[i], out);
      }
    }
    list[i] = {ptr<void>(in), ptr<void>(out), in.numel(), type_of(in, ""), type_of(out, "")};
  }
  const auto options = at::TensorOptions().device(device);
  const Tensor norm = at::empty({}, options.dtype(at::kFloat));
  const size_t bytes = fp8gmm_multi_norm_workspace_bytes((int)list.size());
  const Tensor work = at::empty({(int64_t)bytes}, options.dtype(at::kByte));
  timed("multi_clip", bytes_of(tensors) + bytes_of(outs), [&] {
    const int rc = fp8gmm_multi_clip(list.data(), (int)list.size(), max_norm, ptr<float>(norm), ptr<void>(work), bytes,
                                     current_stream(device));
    TORCH_CHECK(rc != FP8GMM_ERR_BAD_ARGUMENT, "fp8_gmm_amd: a result of multi_clip overlaps another tensor of the call");
    check(rc);
  });
  for (auto& c : copies) c.first.copy_(c.second);
  for (const Tensor& t : outs) torch::autograd::impl::bump_version(t);
  return norm;
}

}  // namespace

void define_layers(py::module_& m) {
  m.def("layer_norm", &layer_norm);
  m.def("rms_norm", [](const Tensor& x, const Tensor& weight, double eps, const std::optional<Tensor>& residual) -> py::object {
    const auto out = rms_norm(x, weight, eps, residual);
    return out.second.defined() ? py::cast(out) : py::cast(out.first);
  });
  m.def("rms_norm_fp8", [](const Tensor& x, const Tensor& weight, double eps, const std::optional<Tensor>& residual,
                           const std::optional<Tensor>& scale, const std::optional<Tensor>& amax, at::ScalarType format) {
    const auto [q, scale_inv, h] = rms_norm_fp8(x, weight, eps, residual, scale, amax, format);
    const auto given = [](const Tensor& t) { return t.defined() ? py::cast(t) : py::object(py::none()); };
    return py::make_tuple(q, given(scale_inv), given(h));
  });
  m.def("embedding", &embedding);
  m.def("multi_norm", &multi_norm);
  m.def("multi_clip", &multi_clip);
}

}  // namespace fp8gmm_host
