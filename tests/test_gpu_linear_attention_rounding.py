"""How far linear attention's results are from 64 bits, as norms: the bounds that its
roundings leave (linear_attention_rounding.py), for decays as slow as long memory needs
(the state carries most of the output) and fast ones, through every kind of pass."""
import pytest
import torch

from oracle import linear_attention_ref as R
from tests import linear_attention_rounding as L

pytestmark = pytest.mark.gpu

SCALE = 0.7
SHAPES = [
    # batch, seq_len, heads, groups, key, value: eight waves and four, segments and one
    (1, 2048, 2, 2, 128, 128), (1, 1100, 2, 2, 64, 64), (2, 130, 3, 3, 32, 48), (1, 700, 2, 2, 24, 128),
    # heads that share keys, every tile size; two heads to a workgroup
    (1, 512, 4, 1, 128, 64), (1, 512, 4, 1, 64, 128), (1, 300, 3, 1, 128, 128), (1, 300, 5, 1, 64, 64),
    (16, 130, 32, 16, 72, 16),
]


def make(b, t, h, grp, kd, vd, dtype, decay, state=3.0, seed=0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    if decay.startswith("slow"):  # 1 - 2^-7 to 1 - 2^-9
        size = (b, t, h) if decay == "slow-token" else (h,)
        g = torch.log1p(-torch.exp2(-7.0 - 2.0 * torch.rand(*size, generator=gen)))
    else:                         # one per token: 1 - 2^-9 to e^-2.7, some that clear the state
        g = -torch.exp(torch.rand(b, t, h, generator=gen) * 7.0 - 6.0)
        if decay == "wild":
            g[torch.rand(b, t, h, generator=gen) < 0.1] = -float("inf")
    return dict(q=r(b, t, grp, kd).to(dtype), k=(r(b, t, grp, kd) * kd ** -0.5).to(dtype),
                v=r(b, t, h, vd).to(dtype), g=g, dout=r(b, t, h, vd).to(dtype),
                h_init=state * r(b, h, kd, vd) if state else None,
                dlast=state * r(b, h, kd, vd) if state else None)


def results(c, dev, requires):
    from ssm_mamba_amd.ops import linear_attention_fn
    x = {n: None if c[n] is None else c[n].to(dev).requires_grad_(n in requires)
         for n in ("q", "k", "v", "g", "h_init")}
    out, last = linear_attention_fn(x["q"], x["k"], x["v"], x["g"], scale=SCALE, h_init=x["h_init"],
                                    return_last_state=True)
    names = [n for n in x if x[n] is not None and x[n].requires_grad]
    outs, gouts = [out], [c["dout"].to(dev)]
    if c["dlast"] is not None:
        outs, gouts = outs + [last], gouts + [c["dlast"].to(dev)]
    grads = torch.autograd.grad(outs, [x[n] for n in names], gouts)
    return dict(out=out, last=last, **{"dinit" if n == "h_init" else "d" + n: d for n, d in zip(names, grads)})


def reference(c):
    args, a = [c[n] for n in "qkvg"], dict(scale=SCALE, h_init=c["h_init"])
    out, last = R.forward(*args, **a)
    return dict(out=out, last=last, **R.backward(*args, c["dout"], dlast=c["dlast"], **a))


def check(got, ref, c, seg=None):
    b, t, h, vd = c["v"].shape
    n = L.chain(c["q"].shape[3], vd, t)
    low = c["v"].dtype == torch.bfloat16
    for name, x in got.items():
        if name == "dg":
            bound = L.bound_decays(*(c[m] for m in "qkvg"), c["dout"], ref, seg, SCALE,
                                   h_init=c["h_init"], dlast=c["dlast"])
        else:
            bound = L.bound_bf16(ref[name], n) if low and name in ("out", "dq", "dk", "dv") else L.bound_fp32(n)
        off = L.relative(x, ref[name])
        print(f"{name}: {off:.3g} of {bound:.3g}")
        assert off <= bound, f"{name}: {off:.4g} off, {bound:.4g} allowed"


def segment(shape, bf16):
    from ssm_mamba_amd import _native
    b, t, h, grp, kd, vd = shape
    chunks = -(-t // L.CHUNK)
    nseg = _native.lib().ssm_linear_attention_segments(b, t, h, grp, kd, vd, int(bf16))
    return -(-chunks // nseg) * L.CHUNK


DTYPES = [torch.bfloat16, torch.float32]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("decay", ["slow", "slow-token", "token", "wild"])
@pytest.mark.parametrize("shape", SHAPES)
def test_every_result(cuda, shape, decay, dtype):
    c = make(*shape, dtype, decay, seed=sum(shape))
    ref = reference(c)
    every = ("q", "k", "v", "g", "h_init")
    if decay.startswith("slow"):
        # the decays' gradient too, which other kernels of dq and dk serve
        check(results(c, cuda, every), ref, c, segment(shape, dtype == torch.bfloat16))
    else:  # its terms there cancel too far for a norm of their own: without it
        check(results(c, cuda, ("q", "k", "v", "h_init")), ref, c)


@pytest.mark.parametrize("shape", SHAPES)
def test_slow_decays_that_need_no_gradient(cuda, shape):
    c = make(*shape, torch.bfloat16, "slow", seed=sum(shape))
    check(results(c, cuda, ("q", "k", "v", "h_init")), reference(c), c)


@pytest.mark.parametrize("shape", [(2, 64, 3, 3, 128, 128), (3, 50, 4, 4, 64, 64), (2, 64, 4, 1, 128, 64),
                                   (1, 33, 6, 2, 40, 72)])
def test_one_chunk_without_a_state(cuda, shape):
    """Nothing but P and the result's own rounding."""
    c = make(*shape, torch.bfloat16, "token", state=0.0, seed=sum(shape))
    check(results(c, cuda, ("q", "k", "v")), reference(c), c)


def test_one_long_segment(cuda):
    """As many heads as fill the machine run their whole sequence in one segment."""
    shape = (64, 513, 8, 8, 16, 24)
    assert segment(shape, True) >= 513
    c = make(*shape, torch.bfloat16, "slow", seed=1)
    check(results(c, cuda, ("q", "k", "v", "g", "h_init")), reference(c), c, 9 * L.CHUNK)
