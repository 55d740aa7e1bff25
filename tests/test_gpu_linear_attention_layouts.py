"""Strided, misaligned and expanded operands in the passes whose heads share keys: the
one that sums over heads, and the one with two heads to a workgroup; padding on either
side, and results that do not depend on how their operands lie in memory."""
import pytest
import torch

from tests.test_gpu_linear_attention import call, check, make

pytestmark = pytest.mark.gpu

# heads that share keys: parts of four heads and of two, tiles of 64 and 128, and (from
# 512 heads on, keys past 64 and values up to 64) two heads to a workgroup
SHAPES = [(2, 150, 6, 2, 64, 64), (1, 200, 7, 1, 128, 64), (1, 200, 4, 1, 40, 128), (2, 130, 6, 3, 128, 96),
          (16, 70, 32, 16, 72, 40), (8, 130, 64, 2, 128, 64)]
DTYPES = [torch.float32, torch.bfloat16]


def layout(kind, c):
    b, t, h, vd = c["v"].shape
    grp, kd = c["q"].shape[2:]
    first = {}

    def wrap(name, x):
        if name == "h_init":
            return x
        if kind == "projection":   # slices of one row: whole 16 bytes where sizes are
            sizes = [grp * kd, grp * kd, h * vd, h]
            if "row" not in first:
                first["row"] = torch.full((b, t, sum(sizes)), float("nan"), dtype=c["v"].dtype, device=x.device)
            if name == "g":
                return x
            i = "qkv".index(name)
            part = first["row"].narrow(-1, sum(sizes[:i]), sizes[i])
            part.copy_(x.flatten(2))
            return part.unflatten(-1, x.shape[2:])
        if kind == "misaligned":   # one element off, odd rows
            n = x.shape[-1]
            wide = torch.full((*x.shape[:-1], n + 9), float("nan"), dtype=x.dtype, device=x.device)
            wide[..., 1:n + 1] = x
            return wide[..., 1:n + 1]
        if kind == "heads first":
            return x.transpose(1, 2).contiguous().transpose(1, 2)
        return x.transpose(0, 1).contiguous().transpose(0, 1)  # tokens first

    return wrap


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["projection", "misaligned", "heads first", "tokens first"])
@pytest.mark.parametrize("shape", SHAPES[:5])
def test_layouts(cuda, shape, kind, dtype):
    c = make(*shape, dtype, seed=sum(shape))
    got = check(c, cuda, dtype, wrap=layout(kind, c))
    x, out, last = call(c, cuda, 0.7)
    names = ("q", "k", "v", "g", "h_init")
    grads = torch.autograd.grad([out, last], [x[n] for n in names], [c["dout"].to(cuda), c["dlast"].to(cuda)])
    for a, b in zip((got[0], got[1], *got[2]), (out, last, *grads)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_expanded_operands(cuda, dtype):
    """One sequence's queries and keys for every row of the batch, and one key for every
    token: strides of zero, whose gradients are sums."""
    from ssm_mamba_amd.ops import linear_attention_fn
    c = make(3, 150, 4, 1, 64, 40, dtype, seed=1, init=False, dlast=False)
    q, k, v, g = (c[n].to(cuda) for n in "qkvg")
    q, k = q[:1].requires_grad_(True), k[:1, :1].requires_grad_(True)
    wide = q.expand(3, 150, 1, 64), k.expand(3, 150, 1, 64)
    got = linear_attention_fn(*wide, v, g, scale=0.7)
    whole = [x.detach().contiguous().requires_grad_(True) for x in wide]
    want = linear_attention_fn(*whole, v, g, scale=0.7)
    assert torch.equal(got, want)
    d = c["dout"].to(cuda)
    a, b = torch.autograd.grad(got, [q, k], d), torch.autograd.grad(want, whole, d)
    # torch's own sums of the same gradients over what was expanded
    assert torch.equal(a[0], b[0].sum(0, keepdim=True))
    assert torch.equal(a[1], b[1].sum((0, 1), keepdim=True))


@pytest.mark.parametrize("side", ["left", "right"])
@pytest.mark.parametrize("shape", SHAPES[1:])
def test_padding_with_shared_heads(cuda, shape, side):
    """Rows of no token, one, some and all; what padding holds is not used."""
    b, t = shape[:2]
    length = ([t // 2, 0, t, 1] * b)[:b]
    c = make(*shape, torch.bfloat16, seed=2, length=length, side=side)
    ref = check(c, cuda, torch.bfloat16)
    at, n = torch.arange(t)[None], c["length"][:, None]
    pad = at >= n if side == "right" else at < t - n
    dirty = dict(c)
    for name in ("q", "k", "v", "dout"):
        dirty[name] = torch.where(pad[..., None, None], torch.tensor(float("nan"), dtype=torch.bfloat16), c[name])
    dirty["g"] = torch.where(pad[..., None], float("nan"), c["g"])
    x, out, last = call(dirty, cuda, 0.7)
    grads = torch.autograd.grad([out, last], [x[n] for n in ("q", "k", "v", "g", "h_init")],
                                [dirty["dout"].to(cuda), c["dlast"].to(cuda)])
    for a, b in zip((out, last, *grads), (ref[0], ref[1], *ref[2])):
        assert torch.equal(a, b)


@pytest.mark.parametrize("shape", [s for s in SHAPES if s[3] > 1])
def test_a_heads_results_do_not_depend_on_its_neighbours(cuda, shape):
    """Each group alone gives the bits that it gives among others."""
    from ssm_mamba_amd import _native
    from ssm_mamba_amd.ops import linear_attention_fn
    b, t, h, grp, kd, vd = shape
    seg = _native.lib().ssm_linear_attention_segments
    assert seg(b, t, h, grp, kd, vd, 1) == seg(b, t, h // grp, 1, kd, vd, 1)  # as long segments
    c = make(*shape, torch.bfloat16, seed=3, init=False)
    q, k, v, g = (c[n].to(cuda) for n in "qkvg")
    with torch.no_grad():
        out = linear_attention_fn(q, k, v, g)
        rep = h // grp
        alone = [linear_attention_fn(q[:, :, i:i + 1], k[:, :, i:i + 1], v[:, :, i * rep:(i + 1) * rep],
                                     g[:, :, i * rep:(i + 1) * rep]) for i in range(grp)]
    assert torch.equal(out, torch.cat(alone, dim=2))
