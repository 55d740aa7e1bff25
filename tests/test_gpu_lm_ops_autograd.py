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
