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


P = 4096  # never dereferenced


def test_more_heads_than_a_launch_holds():
    """512 threads for each of 2^23 heads would be 2^32: refused before any launch."""
    import ctypes

    from ssm_mamba_amd import _native as N
    lib = N.lib()
    b, h = 65535, 129
    assert b * h >= 1 << 23 and 65535 * 128 < 1 << 23
    s = (ctypes.c_int64 * 12)(*[4096, 8, 4] * 4)
    big = 1 << 62
    got = [lib.ssm_linear_attention_fwd(b, 1, h, 1, 4, 4, 0, P, P, P, s, P, 0, 0, 1.0, None, None, 0, P,
                                        None, P, P, big, None),
           lib.ssm_linear_attention_bwd(b, 1, h, 1, 4, 4, 0, P, P, P, P, s, P, 0, 0, 1.0, None, None, 0,
                                        P, None, None, P, P, P, None, None, P, big, None),
           lib.ssm_linear_attention_step(b, h, 1, 4, 4, 0, P, P, P, P, s, P, 0, 1.0, P, None)]
    assert got == [2, 2, 2] and b"batch * heads < 2^23" in lib.ssm_last_error()
    assert lib.ssm_linear_attention_segments(b, 1, h, 1, 4, 4, 0) == 0
    assert lib.ssm_linear_attention_segments(65535, 1, 128, 1, 4, 4, 0) == 1


@pytest.mark.parametrize("tokens", [1 << 20, 1 << 29, (1 << 31) - 65537])
def test_embedding_workspace_of_many_tokens(tokens):
    """(token, position) pairs twice, 128 workgroups' counts of 1024, a run a row and a
    row of sums for 32 positions: up to the most tokens there can be."""
    from ssm_mamba_amd import _native as N
    got = N.lib().ssm_embedding_bwd_workspace_bytes(tokens, 1000, 2)
    want = 2 * 8 * tokens + 128 * 1024 * 4 + 1001 * 16 + -(-tokens // 32) * 2 * 4
    assert want - 128 * 1024 * 4 <= got <= want + 5 * 256


def test_clipping_more_than_a_launch_holds():
    """2^24 chunks of 256 threads, sums that would pass 64 bits, and no sizes at all."""
    import ctypes

    from ssm_mamba_amd import _native as N
    lib = N.lib()
    most = (1 << 24) - 1

    def clip(*sizes):
        n = len(sizes)
        arr = lambda t, *x: (t * n)(*(x * n if len(x) == 1 else x))  # noqa: E731
        s = arr(ctypes.c_int64, *sizes)
        return lib.ssm_grad_clip_workspace_bytes(n, s), lambda: lib.ssm_grad_clip(
            n, arr(ctypes.c_void_p, P), arr(ctypes.c_void_p, 2 * P), s, arr(ctypes.c_int, 0),
            arr(ctypes.c_int, 0), 1.0, P, P, 8, None)

    for sizes in ((most * 16384 + 1,), (1 << 37, 1 << 37), ((1 << 63) - 1,),
                  ((1 << 63) - 1, (1 << 63) - 1, (1 << 63) - 1)):
        need, call = clip(*sizes)
        assert need == 0 and call() == 2 and b"2^24 chunks" in lib.ssm_last_error(), sizes
    need, call = clip(most * 16384)
    assert need == most * 8 + 256 and call() == 1 and b"workspace" in lib.ssm_last_error()
    assert lib.ssm_grad_clip_workspace_bytes(-1, None) == 0
    assert lib.ssm_grad_clip_workspace_bytes(2, None) == 0
    assert lib.ssm_grad_clip_workspace_bytes(0, None) == 256
