"""How far linear attention's results may be from 64 bits as norms, from the roundings
alone, and the same chunks on the CPU with a chosen number of bf16 terms.

Signs of the test's inputs are independent, so errors of independent roundings add as
squares, as the terms of a sum themselves do: a rounding that is off by at most e of
each of its values leaves at most e of the result's norm.
* bf16 results: their own rounding, which is that of the exact result (``own``);
  three operands in two bf16 terms each -- P, a value times its decay in the state, and
  the state -- 2^-16 of each; and float32's sums: own + 3 * 2^-16 + chain * 2^-24.
* float32 results (a last state, the first state's gradient): every term passes at most
  ``chain`` float32 roundings, and three bf16 terms hold float32's bits:
  sqrt(chain) * 2^-24.
* the decays' gradient, by sums of q . dq - k . dk to the end of a token's segment and
  <D, S> there: sqrt(chain) * 2^-24 of the root of the sum of these terms' squares, and
  its own rounding, 2^-24.  One decay for a whole head has the tokens' sum, in which a
  term of a segment is as often as the tokens up to it that it is a term of: its error
  is one, so as many times itself before it is squared."""
import torch

from oracle import linear_attention_ref as R

CHUNK = 64


def chain(key, value, seqlen):
    """Roundings in float32 on a term's way: two inner products, a chunk, the chunks,
    decays and products."""
    return key + value + CHUNK + seqlen // CHUNK + 32


def relative(got, ref):
    got, ref = got.detach().double().cpu(), ref.double()
    return float((got - ref).norm() / ref.norm())


def own(ref):
    """What rounding the exact result to bf16 leaves."""
    return relative(ref.to(torch.bfloat16), ref)


def bound_bf16(ref, n):
    return own(ref) + 3 * 2.0 ** -16 + n * 2.0 ** -24


def bound_fp32(n):
    return n ** 0.5 * 2.0 ** -24


def bound_decays(q, k, v, g, dout, ref, seg, scale, h_init=None, dlast=None):
    """The same for dg, relative to its norm; ``ref``: the oracle's gradients, ``seg``:
    tokens of a segment.  The terms are those of every head's own row."""
    b, t, h, vd = v.shape
    rep = h // q.shape[2]
    if rep > 1:  # each head's own dq and dk
        q, k = (x.repeat_interleave(rep, dim=2) for x in (q, k))
        ref = R.backward(q, k, v, g, dout, scale=scale, h_init=h_init, dlast=dlast)
    flow = ((q.double() * ref["dq"]) ** 2).sum(-1) + ((k.double() * ref["dk"]) ** 2).sum(-1)
    gw = g.expand(b, t, h)
    squares = torch.zeros(h, dtype=torch.float64)
    for t0 in range(0, t, seg):
        t1 = min(t0 + seg, t)
        # how often a token's terms are in the results: at every token up to it, as a
        # square each, or in one sum
        times = torch.arange(1, t1 - t0 + 1, dtype=torch.float64) ** (2 if g.dim() == 1 else 1)
        squares += (flow[:, t0:t1] * times[None, :, None]).sum((0, 1))
        S = R.forward(q[:, :t1], k[:, :t1], v[:, :t1], gw[:, :t1], h_init=h_init)[1]
        D = dlast
        if t1 < t:
            D = R.backward(q[:, t1:], k[:, t1:], v[:, t1:], gw[:, t1:], dout[:, t1:], scale=scale,
                           h_init=S, dlast=dlast)["dinit"]
        if D is not None:
            squares += times[-1] * ((S * D.double()) ** 2).sum((0, 2, 3))
    n = chain(q.shape[3], vd, t)
    return 2.0 ** -24 + bound_fp32(n) * float(squares.sum().sqrt() / ref["dg"].norm())


def _split(x, n):
    out = []
    for _ in range(n):
        out.append(x.to(torch.bfloat16).float())
        x = x - out[-1]
    return out


def run(x, y, z, g, start, p, u, o, scale_out=1.0, r=None):
    """The chunked pass in float32 over (tokens, size) operands of one head: (out, last
    state, row dots with r), P in ``p`` bf16 terms, values times their decay in ``u``
    and the state as an operand in ``o``; g: log decays in front of each row."""
    S = torch.zeros(y.shape[1], z.shape[1]) if start is None else start.float().clone()
    out, dots = torch.zeros(x.shape[0], z.shape[1]), torch.zeros(x.shape[0])
    for t0 in range(0, x.shape[0], CHUNK):
        a = slice(t0, min(t0 + CHUNK, x.shape[0]))
        c = g[a].double().cumsum(0)
        P = ((x[a] @ y[a].t()) * (c[:, None] - c[None]).exp().float() * scale_out).tril()
        state = sum(x[a] @ s for s in _split(S, o)) * (c.exp().float() * scale_out)[:, None]
        out[a] = state + sum(w @ z[a] for w in _split(P, p))
        if r is not None:
            dots[a] = (r[a] * state).sum(-1) + (P * (r[a] @ z[a].t())).sum(-1)
        weighted = z[a] * (c[-1] - c).exp().float()[:, None]
        S = S * c[-1].exp().float() + sum(y[a].t() @ w for w in _split(weighted, u))
    return out, S, dots


def emulate(q, k, v, g, dout, seg, scale, p=2, u=2, o=2, exact=3):
    """Every result of one head, (tokens, size) float32 tensors of bf16 values; the
    decays' gradient with ``exact`` terms."""
    t = q.shape[0]
    segs = [slice(i, min(i + seg, t)) for i in range(0, t, seg)]
    starts = [None]
    for s in segs:
        starts.append(run(q[s], k[s], v[s], g[s], starts[-1], 1, exact, 1)[1])
    back = [None]
    gr = torch.cat([g[1:], torch.zeros(1)])  # in front of each row in reversed time
    for s in reversed(segs):
        back.append(run(*(x[s].flip(0) for x in (k, q, dout * scale, gr)), back[-1], 1, exact, 1)[1])
    back = back[-2::-1]  # what each segment starts from
    T = lambda x: None if x is None else x.t()  # noqa: E731
    names = ("out", "dq", "dk", "dv", "dg")
    res = {n: [] for n in names}
    for i, s in enumerate(segs):
        Q, K, V, G, DO, GR = (x[s] for x in (q, k, v, g, dout, gr))
        f = lambda x: x.flip(0)  # noqa: E731
        res["out"].append(run(Q, K, V, G, starts[i], p, u, o, scale)[0])
        res["dq"].append(run(DO, V, K, G, T(starts[i]), p, u, o, scale)[0])
        row = run(DO, V, K, G, T(starts[i]), p, exact, exact, scale, r=Q)[2]
        B = None if back[i] is None else back[i]
        res["dk"].append(f(run(f(V), f(DO) * scale, f(Q), f(GR), T(B), p, u, o)[0]))
        col = f(run(f(V), f(DO) * scale, f(Q), f(GR), T(B), p, exact, exact, r=f(K))[2])
        res["dv"].append(f(run(f(K), f(Q), f(DO) * scale, f(GR), B, p, u, o)[0]))
        flow = (row.double() - col.double()).flip(0).cumsum(0).flip(0)
        if B is not None:
            flow = flow + float(g[s.stop].exp()) * (starts[i + 1] * B).double().sum()
        res["dg"].append(flow.float())
    res = {n: torch.cat(x) for n, x in res.items()}
    res["last"] = starts[-1]
    for n in ("out", "dq", "dk", "dv"):
        res[n] = res[n].to(torch.bfloat16)
    return res
