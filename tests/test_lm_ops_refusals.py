"""More refusals of the operators around a matrix-valued state that need no GPU."""
import pytest
import torch


def test_a_trace_is_refused():
    """It would keep the result's allocation and not the kernel that fills it."""
    from ssm_mamba_amd.ops import (clip_grad_norm_, embedding_fn, linear_attention_fn,
                                   linear_attention_step)
    ids, w = torch.tensor([1, 2]), torch.zeros(3, 4)
    x, g = torch.zeros(1, 3, 2, 4), torch.zeros(1, 3, 2)
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.ones(3)
    for name, fn, args in (
            ("embedding_fn", lambda t: embedding_fn(ids, t), w),
            ("linear_attention_fn", lambda t: linear_attention_fn(t, t, t, g), x),
            ("linear_attention_step",
             lambda t: linear_attention_step(torch.zeros(1, 2, 4, 4), t, t, t, g[:, 0]), x[:, 0]),
            ("clip_grad_norm_", lambda t: clip_grad_norm_(p, 1.0) + t.sum(), w)):
        with pytest.raises(RuntimeError, match=name + " cannot be traced"):
            torch.jit.trace(fn, args)
