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
gradient (in grad mode one that requires it is refused), and -inf is a decay of zero.  States are (batch, heads, dk, dv) float32.
"""
from __future__ import annotations

from typing import Optional

import torch

from .._ext import _C


def linear_attention_fn(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
                        scale: Optional[float] = None, initial_state: Optional[torch.Tensor] = None,
                        lengths: Optional[torch.Tensor] = None, return_last_state: bool = False):
    """out (batch, seqlen, heads, dv) in q's dtype, differentiable in q, k, v and initial_state.

    scale defaults to dk ** -0.5.  initial_state (batch, heads, dk, dv) float32, default zero.
    lengths (batch,): tokens from lengths[b] on take no part and give zero outputs and gradients.
    With return_last_state also the float32 state after the last token of each row (after
    lengths[b] tokens), differentiable, from which linear_attention_update continues.

    Infinities and NaN: an infinity in q, k, v or a state may come out as a NaN, since operands are split
    into parts.  Tokens are worked on in chunks: a NaN or an infinity in a token's k or v may also
    reach the outputs of up to 127 tokens before it, and in a backward the gradients of up to 127
    tokens on either side.  Other heads and batch rows are not touched."""
    r = _C.linear_attention(q, k, v, log_decay, scale, initial_state, lengths, return_last_state)
    return (r[0], r[1]) if return_last_state else r[0]


def linear_attention_update(state: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                            log_decay: torch.Tensor, scale: Optional[float] = None) -> torch.Tensor:
    """One decode step; `state` (batch, heads, dk, dv) float32 with unit dv stride is updated in place.
    A state whose elements share memory (an expanded one) is refused.

    q, k: (batch, heads, dk); v: (batch, heads, dv), fewer heads as in linear_attention_fn.
    Returns out (batch, heads, dv) in q's dtype.  Not differentiable: in grad mode a state that requires a
    gradient is refused, and a backward through out raises where q, k or v require one; the new state
    has no history.  Autograd counts the update as any in-place change: a backward that needs the
    state as it was before raises."""
    return _C.linear_attention_update(state, q, k, v, log_decay, scale)


__all__ = ["linear_attention_fn", "linear_attention_update"]
