"""Linear attention with a decay for each head, over matrix-valued states
(no counterpart in the reference, whose states are vectors of a channel):
S_t = exp(g_t) S_{t-1} + k_t v_t^T, o_t = scale S_t^T q_t."""
from __future__ import annotations

from typing import Optional

import torch

from .. import _ext as _E


def linear_attention_fn(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, *,
                        scale: float = 1.0, return_last_state: bool = False,
                        h_init: Optional[torch.Tensor] = None,
                        length: Optional[torch.Tensor] = None, padding_side: str = "left"):
    """o_t = scale S_t^T q_t over S_t = exp(g_t) S_{t-1} + k_t v_t^T, returned
    alone or with the last state.

    q, k (batch, seq_len, groups, key); v (batch, seq_len, heads, value), float32
    or bfloat16 (q and k are cast to v's); heads is a multiple of groups, and
    value head h uses query and key head h // (heads / groups).  key, value <= 128.
    g: log decays, (batch, seq_len, heads) or one per head, (heads,); at most 0
    for a decay, -inf clears the state; computed with in float32.
    h_init, and the last state: (batch, heads, key, value) float32.
    length (batch,) int64 with padding_side: padded tokens leave the state as it
    is, their outputs and gradients are zero, and what q, k, v and g hold there
    is not used.

    bfloat16 results are rounded from float32 sums; the last state, and the
    gradients of g and h_init, are as exact as float32 products.  A value that is not
    finite reaches the results that depend on it, and g's gradients at other tokens.

    Rows of adjacent elements that are 16-byte aligned and whole 16 bytes long are
    read in place, whatever their strides; others are copied.  Differentiable once
    in q, k, v, g and h_init: differentiating its gradients (create_graph) raises, as
    forward mode does."""
    res = _E.module("lm_ops").linear_attention(q, k, v, g, float(scale), h_init, length, padding_side,
                                               bool(return_last_state))
    return (res[0], res[1]) if return_last_state else res[0]


def linear_attention_step(state: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                          g: torch.Tensor, *, scale: float = 1.0) -> torch.Tensor:
    """One token of ``linear_attention_fn``: state (batch, heads, key, value)
    float32 is updated in place; q, k (batch, groups, key); v (batch, heads,
    value); g (batch, heads) or (heads,).  Returns out (batch, heads, value).  No
    autograd, as in ``selective_state_update``."""
    return _E.module("lm_ops").linear_attention_step(state, q, k, v, g, float(scale))
