"""The embedding's gradient past what one launch holds, and the sort over every number of
digits and workgroups."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def gradient(ids, dout, vocab):
    from ssm_mamba_amd import _ext
    return _ext.module("lm_ops").embedding_backward(ids, dout, vocab, 1.0, -1)


def test_more_rows_than_a_launch_holds(cuda):
    """2^24 rows of 256 threads each."""
    vocab, dim = (1 << 24) + 3, 129
    ids = torch.tensor([0, vocab - 1, 5, (1 << 24) - 1, 1 << 24, 5, 1 << 20], device=cuda)
    dout = torch.arange(1, 8, device=cuda)[:, None].expand(7, dim).to(torch.bfloat16).contiguous()
    dw = gradient(ids, dout, vocab)
    for row, value in ((0, 1), (vocab - 1, 2), (5, 9), ((1 << 24) - 1, 4), (1 << 24, 5), (1 << 20, 7)):
        assert (dw[row] == value).all(), row
    assert int(dw.count_nonzero()) == 6 * dim


def test_more_tokens_than_a_launch_holds(cuda):
    """2^29 positions are 2^24 pieces of 32.  Whole numbers: exact in float32."""
    n, vocab = (1 << 29) + 77, 1009
    ids = torch.arange(n, device=cuda) % vocab
    dw = gradient(ids, torch.ones(n, 1, device=cuda), vocab)
    want = torch.full((vocab, 1), float(n // vocab), device=cuda)
    want[:n % vocab] += 1
    assert torch.equal(dw, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n, vocab, dim", [
    (33001, 50280, 8),       # 65 workgroups, two digits
    (70001, 70001, 9),       # 92 workgroups (of 768 positions), two digits
    (65536, 1100000, 8),     # 128 workgroups, three digits
    (5000, 1100000, 8),      # 10 workgroups, three digits
    (4096, 1100000, 8), (4097, (1 << 20) - 1, 8), (4097, 1 << 20, 8)])
def test_digits_and_workgroups_of_the_sort(cuda, dtype, n, vocab, dim):
    """Against sums in 64 bits: r positions are r roundings of 2^-24 of the sum of
    absolute values and the scaling's, and a bf16 result's own, half of eps."""
    gen = torch.Generator().manual_seed(n + vocab)
    u = torch.rand(n, generator=gen, dtype=torch.float64)
    ids = (torch.exp(u * math.log(vocab)).long().clamp(1, vocab) - 1) * 7919 % vocab
    dout = torch.randn(n, dim, generator=gen).to(dtype)
    dw = gradient(ids.to(cuda), dout.to(cuda), vocab).double().cpu()
    ref = torch.zeros(vocab, dim, dtype=torch.float64).index_add_(0, ids, dout.double())
    mag = torch.zeros(vocab, dim, dtype=torch.float64).index_add_(0, ids, dout.double().abs())
    bound = (torch.bincount(ids, minlength=vocab)[:, None] + 2) * 2.0 ** -24 * mag
    if dtype == torch.bfloat16:
        bound += torch.finfo(dtype).eps / 2 * ref.abs()
    assert ((dw - ref).abs() <= bound).all()
