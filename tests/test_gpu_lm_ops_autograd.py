"""Linear attention and the embedding under autograd's other modes: what they cannot
differentiate they refuse, and never answer as a constant."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

pytestmark = pytest.mark.gpu


def operands(cuda, seed=0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen).to(cuda)  # noqa: E731
    return dict(q=r(1, 70, 2, 16), k=r(1, 70, 2, 16) / 4, v=r(1, 70, 4, 24), g=-r(1, 70, 4).abs(),
                h_init=r(1, 4, 16, 24))


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("name", ["q", "k", "v", "g", "h_init"])
def test_forward_mode_of_linear_attention_is_refused(cuda, name, grad):
    from ssm_mamba_amd.ops import linear_attention_fn
    x = operands(cuda)
    with torch.set_grad_enabled(grad), fwd.dual_level():
        x[name] = fwd.make_dual(x[name], torch.ones_like(x[name]))
        with pytest.raises(RuntimeError, match="jvp is not implemented"):
            linear_attention_fn(x["q"], x["k"], x["v"], x["g"], h_init=x["h_init"])


@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_of_the_embedding_is_refused(cuda, grad):
    from ssm_mamba_amd.ops import embedding_fn
    w = torch.randn(9, 8, device=cuda)
    with torch.set_grad_enabled(grad), fwd.dual_level():
        with pytest.raises(RuntimeError, match="jvp is not implemented"):
            embedding_fn(torch.tensor([1, 2], device=cuda), fwd.make_dual(w, torch.ones_like(w)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("pad", [None, 3])
def test_second_and_third_derivatives_of_the_embedding(cuda, dtype, pad):
    """Whole numbers, exact in every type: against the same formulas by indexing.  The
    weight's gradient is linear in the output's, so differentiating it gives the lookup
    (no rows for padding), and that gives the sums again."""
    from ssm_mamba_amd.ops import embedding_fn
    vocab, dim = 7, 12
    gen = torch.Generator().manual_seed(0)
    ids = torch.randint(0, vocab, (3, 5), generator=gen)
    whole = lambda *s: torch.randint(-3, 4, s, generator=gen).float()  # noqa: E731
    w, d, a, b = whole(vocab, dim), whole(3, 5, dim), whole(vocab, dim), whole(3, 5, dim)
    keep = (ids != pad).float()[..., None] if pad is not None else torch.ones(3, 5, 1)
    at = ids.to(cuda)
    W, D, A = (x.to(cuda, dtype).requires_grad_(True) for x in (w, d, a))
    dw, = torch.autograd.grad(embedding_fn(at, W, scale=2.0, padding_idx=pad), W, D, create_graph=True)
    sums = lambda x: torch.zeros(vocab, dim).index_add_(0, ids.view(-1), (x * keep).view(-1, dim))  # noqa: E731
    assert torch.equal(dw.detach().float().cpu(), 2 * sums(d))
    dd, = torch.autograd.grad(dw, D, A, create_graph=True)
    assert torch.equal(dd.detach().float().cpu(), 2 * a[ids] * keep)
    da, = torch.autograd.grad(dd, A, b.to(cuda, dtype))
    assert torch.equal(da.float().cpu(), 2 * sums(b))


def test_second_derivative_through_an_embedding(cuda):
    """A penalty on the weight's gradient, as a program has it, against torch's."""
    from ssm_mamba_amd.ops import embedding_fn
    gen = torch.Generator().manual_seed(1)
    w0 = torch.randn(11, 8, generator=gen, dtype=torch.float64)
    ids = torch.randint(0, 11, (20,), generator=gen)

    def penalty(lookup, w):
        g, = torch.autograd.grad(lookup(w).pow(3).sum(), w, create_graph=True)
        return torch.autograd.grad(g.square().sum(), w)[0]

    want = penalty(lambda w: w[ids], w0.clone().requires_grad_(True))
    got = penalty(lambda w: embedding_fn(ids.to(cuda), w), w0.float().to(cuda).requires_grad_(True))
    # sums of up to 20 products of a few roundings each, twice
    assert ((got.double().cpu() - want).abs() <= 64 * 2.0 ** -24 * want.abs() + 1e-30).all()


def test_tokens_outside_the_vocabulary_twice(cuda):
    from ssm_mamba_amd.ops import embedding_fn
    ids = torch.tensor([0, -1, 4, 3], device=cuda)
    w = torch.ones(4, 8, device=cuda, requires_grad=True)
    d = torch.ones(4, 8, device=cuda, requires_grad=True)
    dw, = torch.autograd.grad(embedding_fn(ids, w), w, d, create_graph=True)
    dd, = torch.autograd.grad(dw.sum(), d)
    assert torch.equal(dd[:, 0].cpu(), torch.tensor([1.0, 0.0, 0.0, 1.0]))


@pytest.mark.parametrize("shared", [False, True])
def test_second_derivatives_of_linear_attention_raise(cuda, shared):
    """Its gradients themselves may be had with create_graph, as without."""
    from ssm_mamba_amd.ops import linear_attention_fn
    x = operands(cuda)
    if not shared:
        x["q"], x["k"] = (x[n].repeat_interleave(2, 2) for n in "qk")
    x = {n: t.requires_grad_(True) for n, t in x.items()}
    out, last = linear_attention_fn(x["q"], x["k"], x["v"], x["g"], h_init=x["h_init"],
                                    return_last_state=True)
    loss = out.square().sum() + last.sum()
    want = torch.autograd.grad(loss, list(x.values()), retain_graph=True)
    got = torch.autograd.grad(loss, list(x.values()), create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    for g in got:
        assert g.requires_grad
        with pytest.raises(RuntimeError, match="linear_attention_fn is differentiable once"):
            torch.autograd.grad(g.square().sum(), x["v"], retain_graph=True)
    # one input's gradient alone, and backward() into .grad
    only, = torch.autograd.grad(out.sum(), x["k"], retain_graph=True, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        only.sum().backward(retain_graph=True)
    out.sum().backward()
    assert all(t.grad is not None and not t.grad.requires_grad for t in x.values())


def test_second_derivative_by_the_results_gradient_raises(cuda):
    """Of operands that are copied on their way, too."""
    from ssm_mamba_amd.ops import linear_attention_fn
    x = operands(cuda)
    wide = torch.randn(1, 70, 2, 17, device=cuda, requires_grad=True)
    out = linear_attention_fn(wide[..., 1:], x["k"], x["v"], x["g"])
    d = torch.randn_like(out).requires_grad_(True)
    dq, = torch.autograd.grad(out, wide, d, create_graph=True)
    for to in (d, wide):
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(dq.sum(), to, retain_graph=True, allow_unused=True)
