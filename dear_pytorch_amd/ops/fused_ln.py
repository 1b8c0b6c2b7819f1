"""Fused residual add + layer norm (CDNA4 kernels, csrc/layer_norm.hip).

``layer_norm(x, weight, bias, eps, residual)`` normalises ``x + residual``
over the last axis; ``FusedLayerNorm`` is the module around it, state-dict
compatible with nn.LayerNorm, and what models/bert.py uses with
``BertConfig(fused_ln=True)`` in place of nn.LayerNorm(x + h) (the reference's
BERT benchmark gets its layer norm from transformers,
dear/bert_benchmark.py:72-99).

Types: x and residual are float32, bfloat16 or float16 of one type, or one of
them is float32 and the other 16-bit (the branch and the residual stream of a
model under autocast); the result has the wider type. weight and bias are
float32 or of the result's type. The sum and all statistics are float32, and
autocast does not change them. Any strides; the result is contiguous. The
gradients of x and residual are the same numbers, and the same tensor where
they have the same type. It is differentiable once.

On the CPU the same numbers come from a torch composition; on a GPU the native
extension is required, and forward-mode derivatives and tracing
(torch.jit.trace, make_fx) raise.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn
import torch.nn.functional as F

from .fused import _native

__all__ = ["layer_norm", "FusedLayerNorm"]

_TYPES = (torch.float32, torch.bfloat16, torch.float16)


def _check(x, weight, bias, residual):
    if x.dim() < 1 or not 1 <= x.size(-1) < 1 << 30:
        raise ValueError("layer_norm: x needs a last axis of 1 to 2^30 - 1 "
                         "elements")
    types = _TYPES + (torch.float64,)
    out = x.dtype
    if x.dtype not in types:
        raise TypeError(f"layer_norm: x must be a float tensor, got {x.dtype}")
    if residual is not None:
        if residual.dtype not in types:
            raise TypeError("layer_norm: residual must be a float tensor, "
                            f"got {residual.dtype}")
        if residual.shape != x.shape or residual.device != x.device:
            raise ValueError("layer_norm: the residual needs x's shape and "
                             "device")
        out = torch.promote_types(x.dtype, residual.dtype)
        if out not in (x.dtype, residual.dtype):
            raise TypeError("layer_norm: x and residual are of two 16-bit "
                            "types")
    for t in (weight, bias):
        if t is None:
            continue
        if t.shape != x.shape[-1:] or t.device != x.device \
                or not t.is_contiguous():
            raise ValueError("layer_norm: weight and bias need shape "
                             f"({x.size(-1)},), contiguous, on x's device")
        if t.dtype not in (torch.float32, out):
            raise TypeError("layer_norm: weight and bias are float32 or of "
                            "the result's type")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError("layer_norm: weight and bias are of two types")
    return out


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None,
               bias: Optional[torch.Tensor] = None, eps: float = 1e-5, *,
               residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """(z - mean z) / sqrt(var z + eps) * weight + bias over the last axis,
    z = x + residual, with the biased variance."""
    if not eps >= 0.0:
        raise ValueError(f"layer_norm: eps must not be negative, got {eps}")
    if x.is_cuda:
        return _native().layer_norm(x, weight, bias, eps, residual)
    out = _check(x, weight, bias, residual)
    # 16-bit inputs are computed in float32, as the kernels do
    calc = torch.float64 if out == torch.float64 else torch.float32
    z = x.to(calc)
    if residual is not None:
        z = z + residual.to(calc)
    w = None if weight is None else weight.to(calc)
    b = None if bias is None else bias.to(calc)
    return F.layer_norm(z, x.shape[-1:], w, b, eps).to(out)


class FusedLayerNorm(nn.LayerNorm):
    """nn.LayerNorm over the last axis with an optional fused residual add.

    forward(x, residual=None) computes layer_norm(x + residual).
    """

    def __init__(self, normalized_shape, *args, **kw):
        super().__init__(normalized_shape, *args, **kw)
        if len(self.normalized_shape) != 1:
            raise ValueError("FusedLayerNorm normalises the last axis only, "
                             f"got {tuple(self.normalized_shape)}")

    def forward(self, x, residual: Optional[torch.Tensor] = None):
        if x.shape[-1:] != self.normalized_shape:
            raise ValueError(f"FusedLayerNorm({self.normalized_shape[0]}) got "
                             f"a last axis of {tuple(x.shape[-1:])}")
        return layer_norm(x, self.weight, self.bias, self.eps,
                          residual=residual)
