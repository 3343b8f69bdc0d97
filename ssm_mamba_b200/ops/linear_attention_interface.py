"""Linear attention with a decay for each head: the matrix-state layer that hybrid stacks put
between Mamba layers.  No counterpart in the reference.

Per batch row and head h, with w = exp(log_decay[h]) and a (dk, dv) state S:
    S_t = w S_{t-1} + k_t v_t^T,   out_t = scale * q_t^T S_t
    linear_attention_fn(q, k, v, log_decay, scale=None, initial_state=None, lengths=None,
                        return_last_state=False)      -> out  or  (out, last_state)
    linear_attention_update(state, q, k, v, log_decay, scale=None) -> out, state in place
The first runs whole sequences in chunks (prompts, training); the second is one decode step.

q, k (batch, seqlen, heads, dk), v (batch, seqlen, heads, dv) in float32 or bfloat16 with any
batch, token and head strides (column blocks of one projection need no copy), dk and dv up to
128; q, k and v may have fewer heads than log_decay, each count dividing it (head h reads head
h // (heads / count)).  log_decay (heads,) float32 is a constant of the layer: it has no
gradient, and -inf is a decay of zero.  States are (batch, heads, dk, dv) float32.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from .._ext import _C
from .selective_scan_interface import ensure_contiguous


def _unit_channel_stride(x: torch.Tensor) -> torch.Tensor:
    return x if x.stride(-1) == 1 else x.contiguous()


class LinearAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, scale, initial_state, lengths, return_last_state):
        out, last = _C.linear_attn_fwd(q, k, v, log_decay, scale, initial_state, lengths, return_last_state)
        ctx.save_for_backward(q, k, v, log_decay, initial_state, lengths)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return (out, last) if return_last_state else out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dlast=None):
        q, k, v, log_decay, initial_state, lengths = ctx.saved_tensors
        if dout is None:
            dout = q.new_zeros(q.shape[0], q.shape[1], log_decay.shape[0], v.shape[3])
        dq, dk, dv, dinit = _C.linear_attn_bwd(q, k, v, log_decay, ctx.scale, initial_state, lengths,
                                               _unit_channel_stride(dout), ensure_contiguous(dlast),
                                               ctx.needs_input_grad[5])
        return dq, dk, dv, None, None, dinit, None, None


def _check(name, q, k, v, log_decay):
    if q.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"{name}: q must be float32 or bfloat16, got {q.dtype}")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"{name}: q, k and v must share a dtype, got {q.dtype}, {k.dtype}, {v.dtype}")
    if log_decay.requires_grad:
        raise ValueError(f"{name}: log_decay is a constant of the layer and has no gradient; pass log_decay.detach()")


def linear_attention_fn(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
                        scale: Optional[float] = None, initial_state: Optional[torch.Tensor] = None,
                        lengths: Optional[torch.Tensor] = None, return_last_state: bool = False):
    """out (batch, seqlen, heads, dv) in q's dtype, differentiable in q, k, v and initial_state.

    scale defaults to dk ** -0.5.  initial_state (batch, heads, dk, dv) float32, default zero.
    lengths (batch,): tokens from lengths[b] on take no part and give zero outputs and gradients.
    With return_last_state also the float32 state after the last token of each row (after
    lengths[b] tokens), differentiable, from which linear_attention_update continues."""
    _check("linear_attention_fn", q, k, v, log_decay)
    if lengths is not None:
        lengths = lengths.to(device=q.device, dtype=torch.int64).contiguous()
    if initial_state is not None and initial_state.dtype != torch.float32:
        raise TypeError(f"linear_attention_fn: initial_state must be float32, got {initial_state.dtype}")
    q, k, v = map(_unit_channel_stride, (q, k, v))
    return LinearAttentionFn.apply(q, k, v, log_decay.float().contiguous(),
                                   float(q.shape[-1] ** -0.5 if scale is None else scale),
                                   ensure_contiguous(initial_state), lengths, bool(return_last_state))


def linear_attention_update(state: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                            log_decay: torch.Tensor, scale: Optional[float] = None) -> torch.Tensor:
    """One decode step; `state` (batch, heads, dk, dv) float32 is updated in place.

    q, k: (batch, heads, dk); v: (batch, heads, dv), fewer heads as in linear_attention_fn.
    Returns out (batch, heads, dv) in q's dtype.  Not differentiable."""
    _check("linear_attention_update", q, k, v, log_decay)
    q, k, v = map(_unit_channel_stride, (q, k, v))
    return _C.linear_attn_update(state, q, k, v, log_decay.float().contiguous(),
                                 float(q.shape[-1] ** -0.5 if scale is None else scale))


__all__ = ["LinearAttentionFn", "linear_attention_fn", "linear_attention_update"]
