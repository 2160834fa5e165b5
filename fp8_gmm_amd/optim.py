"""Behind the backward pass: clipping of the gradients by their global norm, and the optimizer's step.

The operand-level calls are ``backend.multi_norm``, ``backend.multi_clip`` and ``backend.multi_adamw``; these are the ones on
parameters, with the names and the arguments that torch's users know.
"""
from itertools import chain

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


def _refuse(options):
    for name in ("amsgrad", "maximize", "differentiable"):
        if options.get(name):
            raise ValueError(f"{name} is not supported")


class AdamW(torch.optim.Optimizer):
    """AdamW with decoupled weight decay, a launch for some dozens of parameters (``backend.multi_adamw``, which has the formulas).

    ``state_bits``: 32, or 8 for moments in ``float8_e4m3fn`` with a float32 scale for every 128 elements, a quarter of the memory.
    ``master_weights``: parameters of 16 bits are copies of float32 masters that the optimizer keeps.  ``max_norm``: every step clips
    the gradients of all groups by their common norm on the way (they stay as they are); the norm before that is ``self.grad_norm``.
    ``capturable``: the steps are counted on the device, a group's for all of its parameters, so that a captured step may be replayed;
    ``lr`` may be a float32 tensor of the device then.  Run one step ahead of the capture: it makes the states.  ``foreach`` and ``fused``,
    which choose one of torch's implementations, choose nothing here; ``amsgrad``, ``maximize`` and ``differentiable`` are refused.

    Parameters are dense, on one device, bfloat16, float16 or float32; those without a gradient are passed over.  Without ``capturable``
    each counts its own steps.  Checkpoints hold the states in their own types, whatever the parameters' (``state_dict``); loading one
    makes new states, of which a graph captured before knows nothing."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, amsgrad=False, *, maximize=False, foreach=None,
                 capturable=False, differentiable=False, fused=None, state_bits=32, master_weights=False, max_norm=None):
        _refuse(dict(amsgrad=amsgrad, maximize=maximize, differentiable=differentiable))
        if state_bits not in (32, 8):
            raise ValueError(f"state_bits must be 32 or 8, got {state_bits}")
        if not (isinstance(lr, torch.Tensor) or lr >= 0.0):
            raise ValueError(f"lr must not be negative, got {lr}")
        if isinstance(lr, torch.Tensor) and not capturable:
            raise ValueError("a tensor for lr needs capturable=True")
        if not all(0.0 <= b < 1.0 for b in betas):
            raise ValueError(f"betas must lie in [0, 1), got {betas}")
        if not (eps >= 0.0 and weight_decay >= 0.0):
            raise ValueError(f"eps and weight_decay must not be negative, got {eps} and {weight_decay}")
        if max_norm is not None and not max_norm >= 0.0:
            raise ValueError(f"max_norm must not be negative, got {max_norm}")
        self.state_bits, self.master_weights, self.max_norm, self.capturable = state_bits, master_weights, max_norm, capturable
        self.grad_norm = None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, steps=None))

    def add_param_group(self, param_group):
        if isinstance(param_group, dict):   # (torch refuses others)
            _refuse(param_group)
        super().add_param_group(param_group)

    def __getstate__(self):   # of a copy or a pickle: the options too, which torch leaves out
        options = ("state_bits", "master_weights", "max_norm", "capturable", "grad_norm")
        return {**super().__getstate__(), **{name: getattr(self, name) for name in options}}

    def _init_state(self, p, state):
        if p.is_cuda and torch.cuda.is_current_stream_capturing():
            _fail("fp8_gmm_amd: a parameter has no state yet: run a step ahead of the capture")
        if not self.capturable:
            state["step"] = 0
        if self.state_bits == 8:
            blocks = -(-p.numel() // 128)
            for moment in ("exp_avg", "exp_avg_sq"):
                state[moment] = torch.zeros_like(p, dtype=torch.float8_e4m3fn)
                state[moment + "_scale"] = torch.zeros(blocks, dtype=torch.float32, device=p.device)
        else:
            for moment in ("exp_avg", "exp_avg_sq"):
                state[moment] = torch.zeros_like(p, dtype=torch.float32)
        if self.master_weights and p.dtype != torch.float32:
            state["master"] = p.detach().float()

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        taken = [[(p, grad) for p in group["params"] if (grad := p.grad) is not None] for group in self.param_groups]
        first = next(chain.from_iterable(taken), (None,))[0]
        if not self.capturable and first is not None and first.is_cuda and torch.cuda.is_current_stream_capturing():
            _fail("fp8_gmm_amd: a captured step needs AdamW(capturable=True): the others' number would be the same in every replay")
        norm = None
        if self.max_norm is not None and first is not None:
            norm = self.grad_norm = backend.multi_norm([grad for _, grad in chain.from_iterable(taken)])
        for group, pairs in zip(self.param_groups, taken):
            if not pairs:
                continue
            calls = {}   # the parameters of a call count the same step, and all have masters or none
            for p, grad in pairs:
                state = self.state[p]
                if not state:
                    self._init_state(p, state)
                calls.setdefault((None if self.capturable else state["step"] + 1, "master" in state), []).append((p, grad, state))
            if self.capturable:
                if group["steps"] is None:
                    group["steps"] = torch.zeros((), dtype=torch.int64, device=pairs[0][0].device)
                group["steps"].add_(1)
            moved = False
            for (step, masters), some in calls.items():
                params, grads, states = zip(*some)

                def of(name):
                    return [state[name] for state in states]

                try:
                    backend.multi_adamw(params, grads, of("exp_avg"), of("exp_avg_sq"), group["steps"] if self.capturable else step,
                                        group["lr"], tuple(group["betas"]), group["eps"], group["weight_decay"],
                                        (of("exp_avg_scale"), of("exp_avg_sq_scale")) if self.state_bits == 8 else None,
                                        of("master") if masters else None, norm, None if norm is None else self.max_norm)
                except Exception:
                    if self.capturable and not moved:   # a step that is refused does not count
                        group["steps"].sub_(1)
                    raise
                moved = True
                if not self.capturable:
                    for state in states:
                        state["step"] = step
        return loss

    def load_state_dict(self, state_dict):
        """A checkpoint of this class and of the same ``state_bits``; its way of counting steps and its masters become this optimizer's."""
        # torch casts the states to their parameters' types: what is loaded, as the caller's hooks ahead of it leave it, is kept to undo
        # that ahead of the hooks behind it.
        loaded = []

        def look(_, state_dict):
            self._check_checkpoint(state_dict)
            loaded.append(state_dict)

        hooks = (self.register_load_state_dict_pre_hook(look),
                 self.register_load_state_dict_post_hook(lambda _: self._take_checkpoint(loaded[0]), prepend=True))
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()

    def _check_checkpoint(self, state_dict):
        for group in state_dict["param_groups"]:
            states = [state_dict["state"][key] for key in group["params"] if key in state_dict["state"]]
            if "steps" not in group or any(("exp_avg_scale" in state) != (self.state_bits == 8) for state in states):
                raise ValueError(f"not a checkpoint of an AdamW of {self.state_bits}-bit moments")
            if self.capturable and len({state.get("step") for state in states}) > 1:
                raise ValueError("the parameters of a capturable group count the same steps, the checkpoint's have different ones")

    def _take_checkpoint(self, state_dict):
        for group, old in zip(self.param_groups, state_dict["param_groups"]):
            device = group["params"][0].device if group["params"] else None
            if isinstance(old["lr"], torch.Tensor):
                group["lr"] = old["lr"].detach().to(device, copy=True) if self.capturable else old["lr"].item()
            steps = old["steps"]
            for key, p in zip(old["params"], group["params"]):
                if key not in state_dict["state"]:
                    continue
                state = self.state[p]
                # torch has cast the tensors to their parameters' types
                state.update((name, value.detach().to(p.device, copy=True))
                             for name, value in state_dict["state"][key].items() if isinstance(value, torch.Tensor))
                if self.capturable:
                    steps = state.pop("step", steps)
                else:
                    state.setdefault("step", None if steps is None else int(steps))
                if not (self.master_weights and p.dtype != torch.float32):
                    state.pop("master", None)
                elif "master" not in state:
                    state["master"] = p.detach().float()
            group["steps"] = torch.full((), int(steps), dtype=torch.int64, device=device) if self.capturable and steps is not None else None
