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

_DTYPES = {torch.float32: _lib.DT_F32, torch.bfloat16: _lib.DT_BF16, torch.float16: _lib.DT_F16}
_KINDS = {1.0: 1, 2.0: 2, math.inf: 0}


def _kind(norm_type) -> int:
    kind = _KINDS.get(float(norm_type))
    if kind is None:
        raise ValueError(f"norm_type is 1, 2 or inf, got {norm_type}")
    return kind


def _gradients(parameters):
    """The gradients of `parameters` (tensors, one tensor, or a generator) that have one, checked."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = [g for g in [p.grad for p in parameters] if g is not None]
    if not grads:
        return grads
    if any(g.layout is not torch.strided for g in grads):
        raise TypeError("gradient norm: sparse gradients are not supported")
    if not {g.dtype for g in grads} <= _DTYPES.keys():
        raise TypeError(f"gradient norm: gradients are fp32, bf16 or fp16, got {sorted(str(g.dtype) for g in grads if g.dtype not in _DTYPES)[0]}")
    if len({g.device for g in grads}) > 1:
        raise ValueError("gradient norm: the gradients are on several devices; combine the norms of each (grad_norm) instead")
    return grads


def _tensor_table(grads):
    table = (_lib.GradTensor * len(grads))()
    for e, g in zip(table, grads):
        e.g, e.n, e.dtype = g.data_ptr(), g.numel(), _DTYPES[g.dtype]
    return table


def _on(device):
    return torch.cuda.device(device) if device.index != torch.cuda.current_device() else _NOTHING


class _Nothing:
    def __enter__(self):
        pass

    def __exit__(self, *a):
        pass


_NOTHING = _Nothing()


def _norm_call(grads, kind, max_norm):
    """(norm before clipping) of contiguous gradients; clips them in place unless max_norm is None."""
    lib = _lib.load()
    dev = grads[0].device
    if dev.type != "cuda":
        raise _lib.CinemaHipError("gradient norm runs HIP kernels: the gradients must live on the GPU")
    table = _tensor_table(grads)
    work = torch.empty(lib.cinema_grad_norm_work_bytes(len(grads)), dtype=torch.uint8, device=dev)
    norm = torch.empty((), dtype=torch.float32, device=dev)
    with _on(dev):
        stream = torch.cuda.current_stream(dev).cuda_stream
        if max_norm is None:
            rc, what = lib.cinema_grad_norm(table, len(grads), kind, work.data_ptr(), norm.data_ptr(), stream), "cinema_grad_norm"
        else:
            rc, what = lib.cinema_grad_clip(table, len(grads), kind, max_norm, work.data_ptr(), norm.data_ptr(), stream), "cinema_grad_clip"
    _lib.check(rc, what)
    return norm


@torch.no_grad()
def grad_norm(parameters, norm_type: float = 2.0):
    """The norm of all gradients of `parameters` taken as one vector: a 0-d fp32 device tensor (no synchronisation); 0 if there
    are none.  norm_type 1, 2 or inf; sums in 64 bits, in a fixed order."""
    kind = _kind(norm_type)
    grads = _gradients(parameters)
    return _norm_call([g.contiguous() for g in grads], kind, None) if grads else torch.zeros(())


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False):
    """torch.nn.utils.clip_grad_norm_: multiplies all gradients by min(1, max_norm / (norm + 1e-6)) in place and returns the
    norm before that (0-d fp32 device tensor).  A norm of at most max_norm writes nothing.  No synchronisation unless
    error_if_nonfinite.  A gradient may not be listed twice or overlap another: they are scaled side by side."""
    kind = _kind(norm_type)
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError(f"max_norm = {max_norm}")
    grads = _gradients(parameters)
    if not grads:
        return torch.zeros(())
    flat = [g if g.is_contiguous() else g.contiguous() for g in grads]
    spans = sorted([(g.data_ptr(), g.data_ptr() + g.numel() * g.element_size()) for g in flat if g.numel()])
    strided = [(g.data_ptr(), g.shape, g.stride()) for g, f in zip(grads, flat) if f is not g]
    if any(a[1] > b[0] for a, b in zip(spans, spans[1:])) or len(set(strided)) < len(strided):
        raise ValueError("clip_grad_norm_: a gradient is listed twice or overlaps another")
    if error_if_nonfinite:
        norm = _norm_call(flat, kind, None)
        if not math.isfinite(float(norm)):
            raise RuntimeError(f"the gradients' norm of order {norm_type} is non-finite ({float(norm)}), so they cannot be clipped")
    norm = _norm_call(flat, kind, max_norm)
    for g, f in zip(grads, flat):
        if f is not g:
            g.copy_(f)
    return norm


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
        """grad_norm: with max_grad_norm, the norm to clip by (0-d fp32 device tensor) in place of this optimiser's own
        gradients' -- for a step whose gradients are spread over several optimisers or processes."""
        entries = []
        for group in self.param_groups:
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.dtype != torch.float32 or not p.is_contiguous() or not p.grad.is_contiguous() or not p.is_cuda:
                    raise _lib.CinemaHipError("HipAdamW needs contiguous fp32 parameters and gradients on the GPU")
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
        norm = None
        if self.max_grad_norm is not None and entries:
            norm = grad_norm
            if norm is None:
                norm = _norm_call([e[2].grad for e in entries], 2, None)
            elif norm.dtype != torch.float32 or norm.numel() != 1 or norm.device != entries[0][1]:
                raise _lib.CinemaHipError("HipAdamW: grad_norm is one fp32 value on the parameters' device")
            self.grad_norm = norm
        for i in range(0, len(entries), _lib.ADAMW_MAX_GROUPS):
            chunk = entries[i:i + _lib.ADAMW_MAX_GROUPS]
            arr = (_lib.AdamWGroup * len(chunk))(*[e[0] for e in chunk])
            stream = C.c_void_p(torch.cuda.current_stream(chunk[0][1]).cuda_stream)
            if norm is not None:
                _lib.check(self._lib.cinema_adamw_step_clipped(arr, len(chunk), int(self.clear_grads), norm.data_ptr(), self.max_grad_norm,
                                                               stream), "cinema_adamw_step_clipped")
                continue
            fn = self._lib.cinema_adamw_step_clear if self.clear_grads else self._lib.cinema_adamw_step
            _lib.check(fn(arr, len(chunk), stream), "cinema_adamw_step")
        return None
