"""The parts of the sequence operators' results that a test has to be able to miss, and limits tight enough for it."""
import torch

from tests import seq_reference as ref

F = 2.0 ** -24
BF, F32 = torch.bfloat16, torch.float32


def attention_limits(want, q, k, v, g, state=None, n=None, dout=None, dstate=None):
    """(name -> d, name -> type) for time-first arguments with heads repeated: a result is off by |round(want) - want| + 2 d at the most.

    A factor of a product on the tensor cores is one bf16 value or the sum of two or three.  Two parts: the first is off by 2^-8 of the
    factor at the most (half a step), the second by 2^-8 of what is left: 2^-16 of the factor.  So held are the pairs' weights (P, E),
    the state before a chunk and its gradient behind it, one of them in a product; k times its decays, three parts, is as good as
    fp32, and so are the factors of fp32 inputs.  Sums are fp32, n terms one after the other: n 2^-24 of the sum of the terms'
    sizes.  With d = (2^-16 + n 2^-24) size a sum is off by d at the most; its rounding to the type is a nearest one, whose
    distance from the grid changes by no more than the sum does."""
    sizes = ref.attention(q.abs(), k.abs(), v.abs(), g, state.abs() if state is not None else None, n, None,
                          dout.abs() if dout is not None else None, dstate.abs() if dstate is not None else None)
    terms, part = q.shape[0] + 2 * max(q.shape[-1], v.shape[-1]) + 24, 2.0 ** -16 if q.dtype == BF else 0.0
    types = {name: F32 if name in ("state", "dstate0") else g.dtype if name == "dg" else q.dtype for name in sizes}
    d = {name: ((0.0 if name in ("state", "dstate0") else part) + terms * F) * size for name, size in sizes.items()}
    if dout is not None:      # the decays' gradient is a running sum of what cancels in a chunk
        qdq, kdk = (q.double().abs() * sizes["dq"]).sum(-1), (k.double().abs() * sizes["dk"]).sum(-1)
        d["dg"] = part * sizes["dg"] + terms * F * (sizes["dg"] + (qdq + kdk).flip(0).cumsum(0).flip(0))
    return d, types


def off_of(x, want, d, kind):
    """How often the limit."""
    return ((x.double() - want).abs() / ((want.to(kind).double() - want).abs() + 2 * d + 1e-30)).max().item()


DECAY_TERMS = ("pairs", "queries of the state", "keys of the state", "state through the chunk")


def decays_gradient(q, k, v, g, state, dout, dstate, chunk, without=None):
    """The gradient of the decays chunk by chunk, in 64 bits, with one of its four terms left out."""
    q, k, v, g, dout = (t.double() for t in (q, k, v, g, dout))
    T, scale = q.shape[0], q.shape[-1] ** -0.5
    S, before, got = state.double(), [], torch.zeros_like(g)
    cuts = [(t, min(t + chunk, T)) for t in range(0, T, chunk)]
    for a, b in cuts:
        before.append(S)
        G = g[a:b].cumsum(0)
        w = (G[-1] - G).exp()[..., None]
        S = G[-1].exp()[..., None, None] * S + torch.einsum("tbhi,tbhj->bhij", k[a:b] * w, v[a:b])
    dS = dstate.double()
    for (a, b), S0 in zip(reversed(cuts), reversed(before)):
        Q, K, V, D, G = q[a:b], k[a:b], v[a:b], dout[a:b], g[a:b].cumsum(0)
        low = torch.ones(b - a, b - a, dtype=torch.bool, device=q.device).tril()[..., None, None]
        M = torch.where(low, (G[:, None] - G[None]).clamp(max=0).exp(), 0.0) * scale * torch.einsum("tbhi,sbhi->tsbh", Q, K) * torch.einsum("tbhj,sbhj->tsbh", D, V)
        pairs = torch.stack([M[t:, :t].sum((0, 1)) for t in range(b - a)])
        queries = (scale * G.exp() * torch.einsum("tbhi,bhij,tbhj->tbh", Q, S0, D)).flip(0).cumsum(0).flip(0)
        keys = (G[-1] - G).exp() * torch.einsum("tbhi,bhij,tbhj->tbh", K, dS, V)
        keys = keys.cumsum(0) - keys
        through = (G[-1].exp() * (S0 * dS).sum((-1, -2))).expand_as(pairs)
        got[a:b] = sum(x for name, x in zip(DECAY_TERMS, (pairs, queries, keys, through)) if name != without)
        dS = G[-1].exp()[..., None, None] * dS + torch.einsum("tbhi,tbhj->bhij", Q * (scale * G.exp())[..., None], D)
    return got


SHORT = [(T, D) for T in (2, 3, 8) for D in ((8, 8), (16, 8), (7, 9))]


def short_state_limit(size, T):
    """Of a state of T tokens, decays of less than 1 in all: T products one after the other, and for each of them the weight (a difference,
    2^x to two units, the scale), its product with k or q and the third part's rounding."""
    return (T + 8) * F * size
