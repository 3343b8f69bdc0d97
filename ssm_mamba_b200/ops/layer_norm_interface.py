"""Layer norm over the last dimension on the sm_100a kernels, with its backward.

    layer_norm_fn(x, weight=None, bias=None, eps=1e-5) -> y
with x (..., dim) in float32 or bfloat16, weight and bias (dim,) or None, y in x's dtype; the
statistics and the sums are float32.  The reference's blocks norm in plain torch (an RMS norm,
nmquan1503/ssm-mamba, modules/rms_norm.py:4-30).
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from .._ext import _C


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x as (rows, dim) with unit element stride: a view where its strides allow."""
    x = x.reshape(-1, x.shape[-1]) if x.numel() else x.reshape(x.shape[:-1].numel(), x.shape[-1])
    return x if x.stride(-1) == 1 else x.contiguous()


class LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        rows = _rows(x)
        y, mean, rstd = _C.layer_norm_fwd(rows, weight, bias, eps, any(ctx.needs_input_grad))
        if mean is not None:
            ctx.save_for_backward(rows, weight, mean, rstd)
            ctx.shape = x.shape
        return y.view(x.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        rows, weight, mean, rstd = ctx.saved_tensors
        dx, dw, db = _C.layer_norm_bwd(rows, weight, mean, rstd, _rows(dy), ctx.needs_input_grad[1],
                                       ctx.needs_input_grad[2])
        return dx.view(ctx.shape), dw, db, None


def layer_norm_fn(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                  eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension, differentiable in
    x, weight and bias."""
    if x.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"layer_norm_fn: x must be float32 or bfloat16, got {x.dtype}")
    if x.dim() < 1:
        raise ValueError("layer_norm_fn: x must have at least one dimension")
    weight, bias = (None if t is None else t.float().contiguous() for t in (weight, bias))
    return LayerNormFn.apply(x, weight, bias, float(eps))


__all__ = ["LayerNormFn", "layer_norm_fn"]
