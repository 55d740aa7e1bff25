"""The bounds on linear attention's roundings accept the terms that its kernels hold and
refuse one term less of any of them (the same chunks emulated on the CPU)."""
import pytest
import torch

from oracle import linear_attention_ref as R
from tests import linear_attention_rounding as L

SCALE = 0.7


def emulated(t, kd, vd, seg, slow, **terms):
    """Each result's distance from 64 bits over its bound."""
    gen = torch.Generator().manual_seed(t)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    q, v, do = (r(t, n).bfloat16().float() for n in (kd, vd, vd))
    k = (r(t, kd) * kd ** -0.5).bfloat16().float()
    g = torch.full((t,), -2.0 ** -8) if slow else -torch.exp(torch.rand(t, generator=gen) * 7 - 6)
    got = L.emulate(q, k, v, g, do, seg, SCALE, **terms)
    one = lambda x: x[None, :, None]  # noqa: E731
    args = [one(x) for x in (q, k, v, g)]
    out, last = R.forward(*args, scale=SCALE)
    ref = dict(out=out, **R.backward(*args, one(do), scale=SCALE))
    n = L.chain(kd, vd, t)
    off = {m: L.relative(one(got[m]), ref[m]) / L.bound_bf16(ref[m], n) for m in ("out", "dq", "dk", "dv")}
    off["last"] = L.relative(got["last"][None, None], last) / L.bound_fp32(n)
    off["dg"] = L.relative(one(got["dg"]), ref["dg"]) / L.bound_decays(*args, one(do), ref, seg, SCALE)
    if slow:  # one decay for the head
        args[3] = g[:1]
        ref = R.backward(*args, one(do), scale=SCALE)
        total = got["dg"].double().sum()[None]
        off["dg of a head"] = L.relative(total.float(), ref["dg"]) / L.bound_decays(*args, one(do), ref, seg, SCALE)
    return off


CASES = [(1100, 128, 128, 128), (1100, 64, 64, 1152), (600, 32, 48, 128)]
BF16 = ("out", "dq", "dk", "dv")


@pytest.mark.parametrize("slow", [False, True])
@pytest.mark.parametrize("case", CASES)
def test_the_kernels_terms_are_within(case, slow):
    off = emulated(*case, slow)
    assert max(off.values()) <= 1, off


@pytest.mark.parametrize("terms, names", [
    (dict(o=1), BF16),                # the state as an operand in one term
    (dict(u=1), BF16),                # values times their decay in one, in the state
    (dict(exact=2), ("last", "dg")),  # two terms where float32's bits are promised
    (dict(exact=1), ("last", "dg"))])
def test_fewer_terms_are_refused(terms, names):
    off = emulated(1100, 64, 64, 1152, True, **terms)
    assert min(off[n] for n in names) > 1, off


@pytest.mark.parametrize("case", CASES + [(64, 128, 128, 64)])
def test_one_term_of_p_is_refused(case):
    off = emulated(*case, False, p=1)
    assert min(off[n] for n in BF16) > 1, off
