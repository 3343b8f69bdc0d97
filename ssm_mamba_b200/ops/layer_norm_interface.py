"""Layer norm over the last dimension on the sm_100a kernels, with its backward.

    layer_norm_fn(x, weight=None, bias=None, eps=1e-5) -> y
with x (..., dim) in float32 or bfloat16, weight and bias (dim,) or None, y in x's dtype; the
statistics and the sums are float32.  The reference's blocks norm in plain torch (an RMS norm,
nmquan1503/ssm-mamba, modules/rms_norm.py:4-30).
"""
from __future__ import annotations

from typing import Optional

import torch

from .._ext import _C


def layer_norm_fn(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                  eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension, differentiable in
    x, weight and bias."""
    return _C.layer_norm(x, weight, bias, eps)


__all__ = ["layer_norm_fn"]
