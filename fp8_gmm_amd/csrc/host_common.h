// What the native host paths share (host_passes.cpp: the grouped modules and the routing; host_layers.cpp: the operators around
// them; host_routing.cpp: the choice of experts; host_adamw.cpp: the optimizer's step).
#pragma once

#include <torch/csrc/autograd/VariableTypeUtils.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/Event.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <c10/hip/HIPStream.h>

#include <atomic>

#include "fp8gmm.h"

namespace fp8gmm_host {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

inline void check(int status) {
  TORCH_CHECK(status == FP8GMM_OK, "fp8gmm error ", status, ": ", fp8gmm_status_string(status));
}

inline void* current_stream(const at::Device& device) {
  return c10::hip::getCurrentHIPStream(device.index()).stream();
}

template <class T>
T* ptr(const Tensor& t) {
  return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}

// An exception of Python code that a pass calls - saved-tensor hooks; activation checkpointing ends its recomputation
// with one - reaches the caller as it is.
template <class F>
Tensor with_python_errors(F&& pass) {
  try {
    return pass();
  } catch (python_error& e) {
    e.restore();
    throw py::error_already_set();
  }
}

// Whether a block of backend.kernel_timing is open (set_kernel_timing).
extern std::atomic<bool> kernel_timing;

// Enqueues what `launch` does; inside a block of kernel_timing between two events, under what `block` makes of the module
// `backend`: a bracket of that block.  On the current device and stream, as the launch.
template <class Block, class Launch>
void timed(Block&& block, Launch&& launch) {
  if (!kernel_timing.load(std::memory_order_relaxed)) return launch();
  py::gil_scoped_acquire gil;
  const py::object bracket = block(py::module_::import("fp8_gmm_amd.backend"));
  bracket.attr("__enter__")();
  launch();
  bracket.attr("__exit__")(py::none(), py::none(), py::none());
}
// ... that moves `bytes` bytes under a name of its own.
template <class Launch>
void timed(const char* name, int64_t bytes, Launch&& launch) {
  timed([&](const py::module_& backend) { return backend.attr("_timed")(name, py::cpp_function([bytes] { return bytes; })); }, launch);
}

// Forward-mode differentiation has no rule here and is refused, as the Python functions refuse it: a tangent that is
// silently dropped would be a wrong derivative.  Under no_grad too, where torch keeps tangents; where it drops them (inference mode)
// none is seen here.  Outside of a level of forward mode there are none to ask the tensors for, which takes a while where they are views.
inline void check_no_tangent(at::TensorList inputs, const char* what = "the grouped modules do") {
  if (torch::autograd::ForwardADLevel::try_get_by_idx(0) == nullptr) return;
  for (const Tensor& t : inputs)
    TORCH_CHECK(!t.defined() || !torch::autograd::isFwGradDefined(t), "fp8_gmm_amd: ", what, " not support forward-mode AD");
}

// The kernels follow addresses: what a transform or a tracer puts in a tensor's place has none.  (A transform under way shows by the
// dispatch key of its layers.)
inline void check_unwrapped(const char* name) {
  TORCH_CHECK(!c10::impl::tls_is_dispatch_key_included(at::DispatchKey::FuncTorchDynamicLayerFrontMode) && !torch::jit::tracer::isTracing(),
              "fp8_gmm_amd: ", name, " does not run under torch.func transforms or tracing");
}

// A gradient as the kernels read it, which see its memory alone: torch hands on such whose sign is a bit beside that, and inside of a
// level of forward mode such with a tangent, which no result of a backward pass here would have.
inline Tensor plain_gradient(const Tensor& grad) {
  check_no_tangent({grad}, "the backward passes do");
  return grad.resolve_neg();
}
// What a backward pass starts from.  A node behind the pass that returned no gradient stands for zeros, as it does for a
// Python autograd function.
inline Tensor gradient_of_result(const Node& node, const variable_list& grads) {
  return grads[0].defined() ? plain_gradient(grads[0]) : node.input_metadata(0).zeros_like();
}

inline int type_of(const Tensor& t, const char* what) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return FP8GMM_TYPE_BF16;
    case at::kHalf: return FP8GMM_TYPE_FP16;
    case at::kFloat: return FP8GMM_TYPE_FP32;
    default: TORCH_CHECK(false, "fp8_gmm_amd: ", what, " must be bfloat16, float16 or float32, got ", t.scalar_type());
  }
}

inline void check_plain(const Tensor& t, const char* what) {
  TORCH_CHECK(t.is_cuda(), "fp8_gmm_amd: expected GPU tensors (the HIP path has no CPU fallback)");
  TORCH_CHECK(t.layout() == at::kStrided && !t.is_neg(), "fp8_gmm_amd: ", what, " must be a dense tensor");
}

inline bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }

// With create_graph the gradients would need a graph of their own, which the kernels do not have: differentiating them again
// raises.  (Left without a node they would pass for constants.)
inline void refuse_second_derivative(variable_list& result, const char* what, at::TensorList inputs) {
  if (!torch::autograd::any_variable_requires_grad({inputs.begin(), inputs.end()})) return;
  auto node = std::shared_ptr<torch::autograd::Error>(
      new torch::autograd::Error(std::string("fp8_gmm_amd: ") + what + " can be differentiated once only",
                                 torch::autograd::collect_next_edges(variable_list(inputs.begin(), inputs.end()))),
      torch::autograd::deleteNode);
  for (Tensor& t : result)
    if (t.defined()) torch::autograd::set_history(t, node);
}

// Memory that a tensor's elements fill without gaps, in whatever order of its dimensions
inline bool dense(const Tensor& t) { return t.is_non_overlapping_and_dense(); }
// The order of the elements in memory, which strides of a dimension of size 1 say nothing of
inline bool same_order(const Tensor& a, const Tensor& b) {
  for (int64_t d = 0; d < a.dim(); ++d)
    if (a.size(d) != 1 && a.stride(d) != b.stride(d)) return false;
  return true;
}
inline bool pass_as_they_are(const Tensor& in, const Tensor& out) { return dense(in) && dense(out) && same_order(in, out); }

void define_layers(py::module_& m);   // host_layers.cpp
void define_routing(py::module_& m);  // host_routing.cpp
void define_adamw(py::module_& m);    // host_adamw.cpp

}  // namespace fp8gmm_host
