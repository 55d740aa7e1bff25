"""Gradients that cannot be scaled in place are refused before anything is written."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def param(grad):
    p = torch.nn.Parameter(torch.zeros(grad.shape, device=grad.device))
    p.grad = grad
    return p


def test_elements_that_share_memory(cuda):
    """An expanded gradient, as autograd hands them out: as an input of `out` it is
    ordinary, in place or as an output it is refused, and the others stay as they were."""
    from ssm_mamba_amd.ops import clip_grad_norm_
    one = torch.full((1,), 2.0, device=cuda)
    ps = [param(torch.full((8,), 3.0, device=cuda)), param(one.expand(10))]
    versions = [p.grad._version for p in ps]
    with pytest.raises(RuntimeError, match="share memory"):
        clip_grad_norm_(ps, 0.5)
    torch.cuda.synchronize()
    assert (ps[0].grad == 3).all() and float(one) == 2.0
    assert [p.grad._version for p in ps] == versions
    out = [torch.empty(8, device=cuda), torch.empty(10, device=cuda)]
    norm = clip_grad_norm_(ps, 0.5, out=out)
    want = (8 * 9.0 + 10 * 4.0) ** 0.5
    # the norm's rounding and the coefficient's: 3 and 4 of 2^-24, the product's one
    assert abs(float(norm) - want) <= 3 * 2.0 ** -24 * want
    for o, v in zip(out, (3.0, 2.0)):
        assert ((o.double() - v * 0.5 / (want + 1e-6)).abs() <= 8 * 2.0 ** -24 * v).all()
    kept = [o.clone() for o in out]
    with pytest.raises(RuntimeError, match="share memory"):
        clip_grad_norm_(ps, 0.25, out=[out[0], one.expand(10)])
    torch.cuda.synchronize()
    assert torch.equal(out[0], kept[0]) and float(one) == 2.0


@pytest.mark.parametrize("into", [False, True])
def test_a_strided_tensor_listed_twice(cuda, into):
    from ssm_mamba_amd.ops import clip_grad_norm_
    wide = torch.ones(6, 9, device=cuda)
    if into:
        ps, out = [param(torch.ones(6, 4, device=cuda)) for _ in "ab"], [wide[:, :4], wide[:, :4]]
    else:
        ps, out = [param(wide[:, :4]), param(wide[:, :4])], None
    with pytest.raises(RuntimeError, match="listed once"):
        clip_grad_norm_(ps, 0.5, out=out)
    torch.cuda.synchronize()
    assert (wide == 1).all()
    # next to each other in one buffer they are two
    ps = [param(wide[:, :4]), param(wide[:, 4:])]
    norm = clip_grad_norm_(ps, 0.5)
    assert abs(float(norm) - 54 ** 0.5) <= 3 * 2.0 ** -24 * 54 ** 0.5
    assert (wide < 0.1).all()
