"""Between the backward pass and the optimizer: clipping of the gradients by their global norm.

The operand-level calls are ``backend.multi_norm`` and ``backend.multi_clip``; this is the one on parameters, with the name and
the arguments that torch's users know.
"""
import torch

from . import backend
from .backend import _fail


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False, foreach=None):
    """Scales the gradients of ``parameters`` (one tensor, or anything that iterates over tensors) in place by ``min(1, max_norm /
    (norm + 1e-6))`` and returns their norm before that, a float32 scalar on their device.  Parameters without a gradient are
    passed over; without any the norm is a zero on the CPU, as torch's.  Gradients are dense, on one device, bfloat16, float16 or
    float32 in any mixture, and none shares memory with another: a parameter that comes twice is refused, not scaled twice.  The norm
    is the 2-norm, summed in float64.  ``foreach`` chooses nothing: there is one way, for all tensors together.
    ``error_if_nonfinite`` waits for the norm and raises ahead of any scaling where it is infinite or a NaN; otherwise such a norm
    makes the gradients zeros or NaN, as torch's call does."""
    if float(norm_type) != 2.0:
        _fail(f"fp8_gmm_amd: clip_grad_norm_ clips by the 2-norm, got norm_type {norm_type}")
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else parameters
    grads = [p.grad for p in parameters if p.grad is not None]
    if not grads:
        return torch.tensor(0.0)
    with torch.no_grad():
        if error_if_nonfinite and not torch.isfinite(norm := backend.multi_norm(grads)):
            _fail(f"fp8_gmm_amd: the norm of the gradients is {norm.item()}")
        return backend.multi_clip(grads, grads, max_norm)
