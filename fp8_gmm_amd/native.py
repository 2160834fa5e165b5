"""The native host path of the modules (csrc/host_passes.cpp) and of the operators around them (csrc/host_layers.cpp,
csrc/host_routing.cpp, csrc/host_adamw.cpp): loads the extension, loudly when it is not built."""
from . import _lib

_lib.load()   # the kernels' library, which the extension calls, with its interface version checked

try:
    from ._host import (Due, Route, Setup, cast_weights, embedding, gating, layer_norm, linear_step, mlp_step, multi_adamw, multi_clip,
                        multi_norm, plain_gradient, rms_norm, rms_norm_fp8, route, select_experts, set_kernel_timing)
except ImportError as exc:
    raise ImportError("fp8_gmm_amd/_host.so is missing or does not load: build the extensions "
                      "(`make -C fp8_gmm_amd/csrc -j8`)") from exc

__all__ = ["Due", "Route", "Setup", "cast_weights", "embedding", "gating", "layer_norm", "linear_step", "mlp_step", "multi_adamw",
           "multi_clip", "multi_norm", "plain_gradient", "rms_norm", "rms_norm_fp8", "route", "select_experts", "set_kernel_timing"]
