"""A residual block with linear attention, as hybrid stacks put between Mamba layers: whole
sequences (training and prompts) and single tokens with an in-place state.

    x       = layer_norm(hidden)
    q, k, v = column blocks of W_qkv x                     (views: nothing is copied)
    o       = linear_attention(q, k, v, log_decay)         a (dk, dv) state per head
    y       = layer_norm(o, per head) * silu(W_gate x)
    out     = hidden + W_out y
The norms, the attention and its decode step are this library's kernels; the projections are plain
GEMMs (torch / cuBLAS).  linear_block_forward with a cache leaves the state that
linear_block_step continues from; the step updates it in place, so it replays from a CUDA graph
(ssm_mamba_b200.decode.GraphedStep).
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch
import torch.nn.functional as F

from .ops import layer_norm_fn, linear_attention_fn, linear_attention_update


@dataclass
class LinearBlockWeights:
    norm_weight: torch.Tensor               # (model,) float32
    norm_bias: torch.Tensor                 # (model,) float32
    qkv_weight: torch.Tensor                # (q_heads * dk + k_heads * dk + v_heads * dv, model)
    gate_weight: torch.Tensor               # (heads * dv, model)
    out_weight: torch.Tensor                # (model, heads * dv)
    log_decay: torch.Tensor                 # (heads,) float32, a constant
    q_heads: int
    k_heads: int
    v_heads: int
    dk: int
    dv: int

    @property
    def heads(self) -> int:
        return self.log_decay.shape[0]

    def split(self, qkv: torch.Tensor):
        q, k, v = qkv.split([self.q_heads * self.dk, self.k_heads * self.dk, self.v_heads * self.dv], dim=-1)
        return (q.unflatten(-1, (self.q_heads, self.dk)), k.unflatten(-1, (self.k_heads, self.dk)),
                v.unflatten(-1, (self.v_heads, self.dv)))


@dataclass
class LinearBlockCache:
    state: torch.Tensor                     # (batch, heads, dk, dv) float32

    @classmethod
    def zeros(cls, w: LinearBlockWeights, batch: int) -> "LinearBlockCache":
        return cls(torch.zeros(batch, w.heads, w.dk, w.dv, dtype=torch.float32, device=w.log_decay.device))


def _finish(w: LinearBlockWeights, hidden: torch.Tensor, x: torch.Tensor, o: torch.Tensor) -> torch.Tensor:
    y = layer_norm_fn(o).flatten(-2) * F.silu(F.linear(x, w.gate_weight))
    return hidden + F.linear(y, w.out_weight)


def linear_block_forward(w: LinearBlockWeights, hidden: torch.Tensor, lengths: Optional[torch.Tensor] = None,
                         cache: Optional[LinearBlockCache] = None) -> torch.Tensor:
    """hidden (batch, seqlen, model) -> (batch, seqlen, model), differentiable.  `lengths`
    (batch,): tokens of each row that count.  With `cache` the sequence continues from its state
    and leaves the state after each row's last token in it.  Gradients stop at the cache: the state it
    brings is a constant, and the one it takes has no history."""
    x = layer_norm_fn(hidden, w.norm_weight, w.norm_bias)
    q, k, v = w.split(F.linear(x, w.qkv_weight))
    if cache is None:
        o = linear_attention_fn(q, k, v, w.log_decay, lengths=lengths)
    else:
        if torch.is_grad_enabled() and cache.state.requires_grad:
            raise ValueError("linear_block_forward: gradients stop at the cache, whose state must not require one")
        # a backward reads the state from before the cache takes the new one
        state = cache.state.clone() if q.requires_grad else cache.state
        o, last = linear_attention_fn(q, k, v, w.log_decay, initial_state=state, lengths=lengths,
                                      return_last_state=True)
        cache.state.copy_(last.detach())
    return _finish(w, hidden, x, o)


def linear_block_step(w: LinearBlockWeights, cache: LinearBlockCache, hidden: torch.Tensor) -> torch.Tensor:
    """One decoding step: hidden (batch, model) -> (batch, model); updates cache.state in place."""
    x = layer_norm_fn(hidden, w.norm_weight, w.norm_bias)
    q, k, v = w.split(F.linear(x, w.qkv_weight))
    return _finish(w, hidden, x, linear_attention_update(cache.state, q, k, v, w.log_decay))


__all__ = ["LinearBlockWeights", "LinearBlockCache", "linear_block_forward", "linear_block_step"]
