"""Embedding lookup with scaling and its weight gradient (the model's
``nn.Embedding``, ``models/causal_lm.py:56``, with a factor on the rows)."""
from __future__ import annotations

from typing import Optional

import torch

from .. import _ext as _E


def embedding_fn(ids: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0,
                 padding_idx: Optional[int] = None) -> torch.Tensor:
    """scale * weight[ids] for ids of any shape (int64 or int32) and weight (vocab,
    dim) float32 or bfloat16, rounded once.  The weight's gradient adds up each
    token's rows in float32 in the order of their positions (the same bits every
    time); row ``padding_idx`` gets none, as in ``torch.nn.Embedding``.  A token
    outside the vocabulary gives NaN and no gradient (no exception: the ids stay
    on the device).  Differentiable any number of times; forward mode is refused."""
    return _E.module("lm_ops").embedding_fn(ids, weight, float(scale), padding_idx)
