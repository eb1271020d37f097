"""The layers of a plain MLP on MI355X, beside the sine layers of models/siren.py: a linear layer whose bias, activation and
residual are part of the product's epilogue, and layer norm, with their gradients (csrc/linear.hip, csrc/layernorm.hip).

Rows are fp32, bf16 or fp16; sums, statistics and epilogues are fp32 inside, results are rounded once.  `LinearAct` and
`LayerNorm` are nn.Linear / nn.LayerNorm as far as constructor, parameters, initialisation and state_dict go.  The reference's
one plain MLP is LatentRegressor (models/inr_decoder.py:126-141).
"""
from __future__ import annotations

import torch.nn as nn

from .. import _lib


def linear_act(x, weight, bias=None, residual=None, activation: str = "none"):
    """act(x W^T + b) + r.  x (..., in), weight (out, in), bias (out,) or None, residual (..., out) or None; activation 'none',
    'relu', 'gelu' (erf), 'gelu_tanh' or 'silu'.  x, weight and residual share a type, the bias may be fp32.  Rows may be
    strided; anything else is made contiguous first.  Under torch.autocast x, weight and residual are cast to its type, an
    fp32 bias stays.  First-order gradients for all four; with a gradient wanted, x, W and the pre-activations (2 bytes each
    for 16-bit rows, 4 for fp32 and where they are few; none without an activation) are kept.  A call that is captured into a
    HIP graph with a gradient wanted is refused while an eager graph of the default stream still uses the same leaves; so is a
    call under torch.jit.trace or make_fx, whose program would not have the launch."""
    return _lib.binding().linear_act(x, weight, bias, residual, activation)


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5):
    """(x - mean) / sqrt(variance + eps) * w + b over the last dimension.  weight and bias (D,) share a type, x's or fp32; each
    may be None.  The result has x's type; under torch.autocast the rows are taken as fp32, as torch does.  First-order
    gradients; with a gradient wanted, x and two fp32 values per row are kept.  Captures and tracing as for linear_act."""
    return _lib.binding().layer_norm(x, weight, bias, eps)


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
