"""Muon: momentum whose matrices are orthogonalised before they are taken from the parameters.

No counterpart in the reference; constructor arguments, state (``momentum_buffer``) and
learning-rate rules are those of ``torch.optim.Muon``. Parameters may also be batches of matrices
[B, ..., M, N] (the SH bands of N splats, [N, 15, 3], are N matrices), and ``step`` takes
the visibility mask of ``SelectiveAdam`` for them. Each parameter group is one call of ``gsb_muon``, in which the parameters
of one shape and type go through the kernels together; those of a group are on one device.
"""

import math

import torch

from ..cuda._wrapper import MUON_COEFFICIENTS, muon


class Muon(torch.optim.Optimizer):
    """``adjust_lr_fn`` scales the update by the matrix's shape: None or ``"original"``:
    sqrt(max(1, M / N)); ``"match_rms_adamw"``: 0.2 sqrt(max(M, N)), the root mean square of an Adam step. The weight
    decay goes by the learning rate alone: param (1 - lr weight_decay).
    ``momentum_dtype``: the type of the momentum buffers (None: the parameter's; or torch.float32).

    bfloat16 parameters with a side above 128 have their updates orthogonalised with 11 significand bits in the products (off
    by up to 0.001 of the update's norm), all others with 22."""

    def __init__(self, params, lr=1e-3, weight_decay=0.1, momentum=0.95, nesterov=True,
                 ns_coefficients=MUON_COEFFICIENTS, eps=1e-7, ns_steps=5, adjust_lr_fn=None, momentum_dtype=None):
        if lr < 0.0 or weight_decay < 0.0:
            raise ValueError(f"lr and weight_decay must not be negative, got {lr}, {weight_decay}")
        if adjust_lr_fn not in (None, "original", "match_rms_adamw"):
            raise ValueError(f"adjust_lr_fn must be None, 'original' or 'match_rms_adamw', got {adjust_lr_fn!r}")
        defaults = dict(lr=lr, weight_decay=weight_decay, momentum=momentum, nesterov=nesterov,
                        ns_coefficients=ns_coefficients, eps=eps, ns_steps=ns_steps, adjust_lr_fn=adjust_lr_fn,
                        momentum_dtype=momentum_dtype)
        super().__init__(params, defaults)

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        try:
            _check_group(self.param_groups[-1])
        except (TypeError, ValueError):
            self.param_groups.pop()
            raise

    def load_state_dict(self, state_dict):
        """As torch's, which casts all state to the parameter's type; the momentum buffers are taken from the saved state
        again, in the group's ``momentum_dtype``. A state of ``torch.optim.Muon`` has none: this optimizer's stays."""
        loaded = []
        hook = self.register_load_state_dict_pre_hook(lambda _, state: loaded.append(state))  # sees what earlier hooks return
        try:
            super().load_state_dict(state_dict)
        finally:
            hook.remove()
        for group, saved in zip(self.param_groups, loaded[-1]["param_groups"]):
            group.setdefault("momentum_dtype", self.defaults["momentum_dtype"])
            for p, key in zip(group["params"], saved["params"]):
                buffer = loaded[-1]["state"].get(key, {}).get("momentum_buffer")
                if buffer is not None:
                    self.state[p]["momentum_buffer"] = buffer.to(p.device, _momentum_type(group, p)).contiguous()

    @torch.no_grad()
    def step(self, visibility=None, closure=None):
        """One step. ``visibility`` [B]: the rows that are stepped, of parameters [B, ..., M, N]. A ``closure`` (also as the only
        argument, as of torch's optimizers) is called first, with gradients on, and its value returned."""
        if callable(visibility):
            if closure is not None:
                raise TypeError("step() takes one closure")
            visibility, closure = None, visibility
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if visibility is not None:
            visibility = visibility.contiguous()
            for group in self.param_groups:  # all or nothing
                for p in group["params"]:
                    if p.grad is not None and (p.dim() < 3 or p.shape[0] != len(visibility)):
                        raise ValueError(f"visibility [{len(visibility)}] does not mask the leading dimension of {tuple(p.shape)}")
        for group in self.param_groups:
            params, grads, buffers, scales = [], [], [], []
            for p in group["params"]:
                if p.grad is None:
                    continue
                state = self.state[p]
                if "momentum_buffer" not in state:
                    state["momentum_buffer"] = torch.zeros_like(p, dtype=_momentum_type(group, p),
                                                                memory_format=torch.contiguous_format)
                grad = p.grad
                if grad.is_sparse:
                    grad = grad.to_dense()
                params.append(p)
                grads.append(grad.contiguous())
                buffers.append(state["momentum_buffer"])
                scales.append(_shape_factor(group["adjust_lr_fn"], *p.shape[-2:]))
            muon(params, grads, buffers, visibility, group["lr"], group["momentum"], group["weight_decay"], group["nesterov"],
                 group["ns_steps"], group["ns_coefficients"], group["eps"], scales)
        return loss


def _check_group(group) -> None:
    for p in group["params"]:
        if p.dim() < 2:
            raise ValueError(f"Muon takes matrices [..., M, N], got a parameter {tuple(p.shape)}")
        if group["momentum_dtype"] not in (None, p.dtype, torch.float32):
            raise TypeError(f"momentum_dtype must be None, the parameter's type or float32, got {group['momentum_dtype']} "
                            f"for {p.dtype}")


def _momentum_type(group, p):
    """The group's, or the parameter's where that does not suit it (a loaded group of parameters of another type)."""
    return group["momentum_dtype"] if group["momentum_dtype"] in (p.dtype, torch.float32) else p.dtype


def _shape_factor(rule, rows: int, cols: int) -> float:
    if rule == "match_rms_adamw":
        return 0.2 * math.sqrt(max(rows, cols))
    return math.sqrt(max(1.0, rows / cols)) if cols else 1.0
