"""Linear attention with a fixed decay for each head.

    S_t = exp(log_decay[h]) S_{t-1} + k_t v_t'        the state of a head, key_dim x value_dim, in 32 bits
    out_t = scale * q_t S_t

`decayed_attention` takes whole sequences (prompts, training) and is differentiable, `decayed_attention_step` a token for each
row.  float32, bfloat16 and float16 CUDA tensors, heads of up to 128 elements.  q, k and v may each have fewer heads than `log_decay`: a number that
divides it, each head then serving several neighbours.  Any strides but a last dimension of neighbouring elements (others are copied).
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _cabi as cabi


def decayed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, *, state: Optional[torch.Tensor] = None,
                      lengths: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(out, final state).  q [batch, tokens, heads, key_dim], k, v [.., value_dim] of one type; out [batch, tokens, heads of log_decay,
    value_dim] in it.  log_decay float32 [heads], at most 0 (-inf: no memory), a constant: it has no gradient.  `state` float32 [batch, heads, key_dim,
    value_dim] is where the sequences go on from (zeros without it).  With `lengths` (integers [batch], on the device) row b has
    lengths[b] tokens: what lies behind them is not used, its outputs and gradients are zero, and the final state is the one after the
    last token.  `scale` is key_dim ** -0.5 unless given.  A value that is not finite reaches no token in front of its own; from there on what it
    reaches is not finite.  Differentiable in q, k, v and state, once; not under a trace."""
    return tuple(cabi.load_binding().decayed_attention(q, k, v, log_decay, state, lengths, q.shape[-1] ** -0.5 if scale is None else scale))


def decayed_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, state: torch.Tensor, *,
                           new_state: Optional[torch.Tensor] = None, active: Optional[torch.Tensor] = None,
                           scale: Optional[float] = None) -> torch.Tensor:
    """One token for each row: q [batch, heads, key_dim] and so on, returns out [batch, heads, value_dim].  The state after the token goes to
    `new_state` (contiguous; `state` itself without it, which is then updated in place).  Rows with active[b] == 0 keep their state and get
    zeros.  No gradient."""
    return cabi.load_binding().decayed_attention_step(q, k, v, log_decay, state, state if new_state is None else new_state, active,
                                                      q.shape[-1] ** -0.5 if scale is None else scale)
