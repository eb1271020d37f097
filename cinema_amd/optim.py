"""AdamW for the hot loop: a torch.optim.Optimizer whose step() is ONE HIP launch over all parameter
groups (cinema_adamw_step).  Same update rule and defaults as torch.optim.AdamW, which the reference
uses (build_atlas.py:453); torch LR schedulers (CosineAnnealingLR, build_atlas.py:455-457) work on it.
Parameters must be contiguous fp32 device tensors.

clip_grad_norm_ / grad_norm: the global norm of many gradients, and torch.nn.utils.clip_grad_norm_, in two launches per 96
tensors (csrc/gradnorm.hip); HipAdamW(max_grad_norm=...) folds the clipping into the update."""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import _lib


def _norm(parameters, norm_type, max_norm):
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    grads = [g for g in [p.grad for p in parameters] if g is not None]
    norm = _lib.binding().grad_norm(grads, norm_type, max_norm)
    return norm if grads or not parameters else norm.new_zeros((), device=parameters[0].device)


def grad_norm(parameters, norm_type: float = 2.0):
    """The norm of all gradients of `parameters` (tensors with .grad, or one) taken as one vector: a 0-d fp32 device tensor, no
    synchronisation; 0 if there are no gradients (on the CPU without any parameters).  norm_type 1, 2 or inf; sums in 64 bits, in
    a fixed order."""
    return _norm(parameters, norm_type, None)


def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False):
    """torch.nn.utils.clip_grad_norm_: multiplies all gradients by min(1, max_norm / (norm + 1e-6)) in place and returns the
    norm before that (0-d fp32 device tensor).  A norm of at most max_norm writes nothing.  No synchronisation unless
    error_if_nonfinite.  A gradient may not be listed twice or overlap another: they are scaled side by side."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    if error_if_nonfinite:
        norm = float(_norm(parameters, norm_type, None))
        if not math.isfinite(norm):
            raise RuntimeError(f"the gradients' norm of order {norm_type} is non-finite ({norm}), so they cannot be clipped")
    return _norm(parameters, norm_type, max_norm)


class HipAdamW(torch.optim.Optimizer):
    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, clear_grads=False,
                 max_grad_norm=None):
        """clear_grads: step() leaves the gradients zeroed (step + the next zero_grad in one pass over them).
        max_grad_norm: step() updates with the gradients of all groups clipped to this 2-norm, as clip_grad_norm_ before it
        would, without writing them; `grad_norm` is then the last step's norm (0-d device tensor)."""
        if max_grad_norm is not None and not float(max_grad_norm) >= 0:
            raise ValueError(f"max_grad_norm = {max_grad_norm}")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        self._lib = _lib.load()
        self.clear_grads = bool(clear_grads)
        self.max_grad_norm = None if max_grad_norm is None else float(max_grad_norm)
        self.grad_norm = None

    @torch.no_grad()
    def step(self, closure=None, grad_norm=None):
        """grad_norm: with max_grad_norm, the norm to clip by (0-d fp32 or fp64 device tensor) in place of this optimiser's own
        gradients' -- for a step whose gradients are spread over several optimisers or processes.  fp32 ends at 3.4e38, and an
        infinite norm makes every gradient zero."""
        if grad_norm is not None:
            if self.max_grad_norm is None:
                raise ValueError("HipAdamW: grad_norm is for an optimiser with max_grad_norm")
            if grad_norm.dtype not in (torch.float32, torch.float64) or grad_norm.numel() != 1 or not grad_norm.is_cuda or any(
                    p.device != grad_norm.device for g in self.param_groups for p in g["params"] if p.grad is not None):
                raise _lib.CinemaHipError("HipAdamW: grad_norm is one fp32 or fp64 value on the parameters' device, a GPU")
        todo = [(group, p) for group in self.param_groups for p in group["params"] if p.grad is not None]
        # whatever can be refused is refused before any state changes
        for _, p in todo:
            if p.dtype != torch.float32 or not p.is_contiguous() or not p.grad.is_contiguous() or not p.is_cuda:
                raise _lib.CinemaHipError("HipAdamW needs contiguous fp32 parameters and gradients on the GPU")
        norm = None
        if self.max_grad_norm is not None and todo:
            self.grad_norm, norm = _lib.binding().grad_norm_wide([p.grad for _, p in todo], 2.0) if grad_norm is None else (grad_norm.float(), grad_norm)
        entries = []
        for group, p in todo:
            st = self.state[p]
            if not st:
                st["step"] = 0
                st["exp_avg"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
                st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
            st["step"] += 1
            g = _lib.AdamWGroup()
            g.p, g.g, g.m, g.v = p.data_ptr(), p.grad.data_ptr(), st["exp_avg"].data_ptr(), st["exp_avg_sq"].data_ptr()
            g.n = p.numel()
            g.lr, (g.beta1, g.beta2) = float(group["lr"]), group["betas"]
            g.eps, g.weight_decay, g.step = float(group["eps"]), float(group["weight_decay"]), int(st["step"])
            entries.append((g, p.device, p))
        for i in range(0, len(entries), _lib.ADAMW_MAX_GROUPS):
            chunk = entries[i:i + _lib.ADAMW_MAX_GROUPS]
            arr = (_lib.AdamWGroup * len(chunk))(*[e[0] for e in chunk])
            stream = C.c_void_p(torch.cuda.current_stream(chunk[0][1]).cuda_stream)
            if norm is not None:
                fn = self._lib.cinema_adamw_step_clipped_f64 if norm.dtype == torch.float64 else self._lib.cinema_adamw_step_clipped
                _lib.check(fn(arr, len(chunk), int(self.clear_grads), norm.data_ptr(), self.max_grad_norm, stream), "cinema_adamw_step_clipped")
                continue
            fn = self._lib.cinema_adamw_step_clear if self.clear_grads else self._lib.cinema_adamw_step
            _lib.check(fn(arr, len(chunk), stream), "cinema_adamw_step")
        return None
