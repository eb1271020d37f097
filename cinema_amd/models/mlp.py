"""The layers of a plain MLP on MI355X, beside the sine layers of models/siren.py: a linear layer whose bias, activation and
residual are part of the product's epilogue, and layer norm, with their gradients (csrc/linear.hip, csrc/layernorm.hip).

Rows are fp32, bf16 or fp16; sums, statistics and epilogues are fp32 inside, results are rounded once.  `LinearAct` and
`LayerNorm` are nn.Linear / nn.LayerNorm as far as constructor, parameters, initialisation and state_dict go.  The reference's
one plain MLP is LatentRegressor (models/inr_decoder.py:126-141).
"""
from __future__ import annotations

import torch
import torch.nn as nn

from .. import _lib
from ..functions import DTYPES, LayerNormFunction, LinearActFunction, layer_norm_forward, linear_act_forward


def _check(what: str, x, like, others):
    """x: the rows; like: name -> tensor (or None) that must have x's type; others: name -> tensor that may also be fp32."""
    if x.dtype not in DTYPES:
        raise TypeError(f"{what}: rows are fp32, bf16 or fp16, got {x.dtype}")
    for name, t in {**like, **others}.items():
        if t is None:
            continue
        if t.device != x.device:
            raise ValueError(f"{what}: {name} is on {t.device}, the rows are on {x.device}")
        if t.dtype != x.dtype and (name in like or t.dtype != torch.float32):
            raise TypeError(f"{what}: {name} has type {t.dtype}, the rows {x.dtype}" + ("" if name in like else " (it may be fp32)"))


def _check_gpu(what: str, x):
    if not x.is_cuda:
        raise RuntimeError(f"cinema_amd {what} runs HIP kernels: the input must live on the GPU")


def linear_act(x, weight, bias=None, residual=None, activation: str = "none"):
    """act(x W^T + b) + r.  x (..., in), weight (out, in), bias (out,) or None, residual (..., out) or None; activation 'none',
    'relu', 'gelu' (erf), 'gelu_tanh' or 'silu'.  x, weight and residual share a type, the bias may be fp32.  Rows may be
    strided; anything else is made contiguous first.  Under torch.autocast x, weight and residual are cast to its type."""
    act = _lib.ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"linear_act: unknown activation {activation!r}, choose from {sorted(_lib.ACTIVATIONS)}")
    if torch.is_autocast_enabled("cuda") and x.is_cuda:
        t = torch.get_autocast_dtype("cuda")
        x, weight = x.to(t), weight.to(t)
        residual = None if residual is None else residual.to(t)
        bias = bias if bias is None or bias.dtype == torch.float32 else bias.to(t)
    _check("linear_act", x, {"weight": weight, "residual": residual}, {"bias": bias})
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1] or weight.numel() == 0:
        raise ValueError(f"linear_act: rows {tuple(x.shape)} do not fit a weight {tuple(weight.shape)}")
    n, k = weight.shape
    lead = x.shape[:-1]
    if bias is not None and bias.shape != (n,):
        raise ValueError(f"linear_act: bias {tuple(bias.shape)} for {n} outputs")
    if residual is not None and residual.shape != lead + (n,):
        raise ValueError(f"linear_act: residual {tuple(residual.shape)} for an output of {tuple(lead) + (n,)}")
    _check_gpu("linear_act", x)
    x2 = x.reshape(-1, k)
    w = weight.contiguous()
    b = None if bias is None else bias.contiguous()
    r2 = None if residual is None else residual.reshape(-1, n)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad) or
                                    (residual is not None and residual.requires_grad)):
        y = LinearActFunction.apply(x2, w, b, r2, act)
    else:
        y, _ = linear_act_forward(x2, w, b, r2, act, False)
    return y.view(lead + (n,))


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5):
    """(x - mean) / sqrt(variance + eps) * w + b over the last dimension.  weight and bias (D,) share a type, x's or fp32; each
    may be None.  The result has x's type; under torch.autocast the rows are taken as fp32, as torch does."""
    if torch.is_autocast_enabled("cuda") and x.is_cuda:
        x = x.float()
        weight = None if weight is None else weight.float()
        bias = None if bias is None else bias.float()
    _check("layer_norm", x, {}, {"weight": weight, "bias": bias})
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"layer_norm: rows {tuple(x.shape)} have no values")
    d = x.shape[-1]
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and t.shape != (d,):
            raise ValueError(f"layer_norm: {name} {tuple(t.shape)} for rows of {d}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"layer_norm: weight is {weight.dtype}, bias {bias.dtype}")
    if not eps >= 0:
        raise ValueError(f"layer_norm: eps = {eps}")
    _check_gpu("layer_norm", x)
    x2 = x.reshape(-1, d)
    w = None if weight is None else weight.contiguous()
    b = None if bias is None else bias.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or (bias is not None and bias.requires_grad)):
        y = LayerNormFunction.apply(x2, w, b, float(eps))
    else:
        y = layer_norm_forward(x2, w, b, float(eps), False)[0]
    return y.view(x.shape)


class LinearAct(nn.Linear):
    """nn.Linear with an activation and an optional residual in the same launch: forward(x, residual=None)."""

    def __init__(self, in_features, out_features, bias=True, activation: str = "none", device=None, dtype=None):
        if activation not in _lib.ACTIVATIONS:
            raise ValueError(f"LinearAct: unknown activation {activation!r}, choose from {sorted(_lib.ACTIVATIONS)}")
        super().__init__(in_features, out_features, bias=bias, device=device, dtype=dtype)
        self.activation = activation

    def forward(self, x, residual=None):
        return linear_act(x, self.weight, self.bias, residual, self.activation)

    def extra_repr(self):
        return super().extra_repr() + f", activation={self.activation!r}"


class LayerNorm(nn.LayerNorm):
    """nn.LayerNorm over the last dimension."""

    def __init__(self, normalized_shape, eps=1e-5, elementwise_affine=True, bias=True, device=None, dtype=None):
        super().__init__(normalized_shape, eps=eps, elementwise_affine=elementwise_affine, bias=bias, device=device, dtype=dtype)
        if len(self.normalized_shape) != 1:
            raise NotImplementedError("cinema_amd LayerNorm normalises over the last dimension only")

    def forward(self, x):
        if x.shape[-1] != self.normalized_shape[0]:
            raise ValueError(f"LayerNorm: rows of {x.shape[-1]} for a norm over {self.normalized_shape[0]}")
        return layer_norm(x, self.weight, self.bias, self.eps)
