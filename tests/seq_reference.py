"""Plain 64-bit forms of the sequence operators, token by token, and bounds of what rounding may do to them.

Every value of the attention is a sum of products.  The same recurrence over absolute values gives, for each result, the sum
of its terms' sizes; a relative error u of some factor moves the result by at most u times that sum."""
import torch

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def attention(q, k, v, g, state=None, lengths=None, scale=None, dout=None, dstate=None):
    """[T, B, H, D] tensors (shared heads already repeated) in float64 -> dict of results."""
    q, k, v, g = (t.double() for t in (q, k, v, g))
    T, B, H, Dk = q.shape
    Dv, dev = v.shape[-1], q.device
    scale = Dk ** -0.5 if scale is None else scale
    S = state.double() if state is not None else torch.zeros(B, H, Dk, Dv, dtype=torch.float64, device=dev)
    n = lengths.clamp(0, T) if lengths is not None else torch.full((B,), T, device=dev)
    out, states = torch.zeros(T, B, H, Dv, dtype=torch.float64, device=dev), [S]
    for t in range(T):
        on = (t < n)[:, None, None, None]
        S = torch.where(on, g[t].exp()[..., None, None] * S + k[t][..., :, None] * v[t][..., None, :], S)
        out[t] = torch.where(on[..., 0], scale * (q[t][..., None, :] @ S).squeeze(-2), 0.0)
        states.append(S)
    r = {"out": out, "state": S}
    if dout is None:
        return r
    dS = dstate.double() if dstate is not None else torch.zeros_like(S)
    dq, dk, dv, dg = (torch.zeros_like(x) for x in (q, k, v, g))
    for t in reversed(range(T)):
        on = (t < n)[:, None, None]
        do = torch.where(on, scale * dout[t].double(), 0.0)
        dS = torch.where(on[..., None], dS + torch.where(on, q[t], 0.0)[..., :, None] * do[..., None, :], dS)
        dq[t] = torch.where(on, (states[t + 1] @ do[..., :, None]).squeeze(-1), 0.0)
        dk[t] = torch.where(on, (dS @ v[t][..., :, None]).squeeze(-1), 0.0)
        dv[t] = torch.where(on, (k[t][..., None, :] @ dS).squeeze(-2), 0.0)
        dg[t] = torch.where(on[..., 0], g[t].exp() * (dS * states[t]).sum((-1, -2)), 0.0)
        dS = torch.where(on[..., None], g[t].exp()[..., None, None] * dS, dS)
    r.update(dq=dq, dk=dk, dv=dv, dg=dg, dstate0=dS)
    return r


def attention_bounds(want, q, k, v, g, state=None, lengths=None, scale=None, dout=None, dstate=None):
    """How far each result may be off.  The type's own rounding of the result, and inside: a factor of a sum that goes to
    the tensor cores is rounded to the type (pairs' weights, the state before a chunk, its gradient: one of them in a
    product, at most two in what a decay moves), everything else is fp32, whose sums have at most n terms
    one after the other.  A factor of an fp32 product is held as two tf32 values of 11 bits: the first is off by 2^-11 at the
    most, and the rest has a bit more than the second can hold, so the factor is off by 2^-23 <= 2^-22; the product of the two small
    halves, 2^-22 of the whole, is left out: 3 * 2^-22 = 12 f a product.  Every result is a sum of products at most two deep (q k, then v): 24 f."""
    u = U[q.dtype]
    neg = None if scale is None else abs(scale)
    sizes = attention(q.abs(), k.abs(), v.abs(), g, state.abs() if state is not None else None, lengths, neg,
                      dout.abs() if dout is not None else None, dstate.abs() if dstate is not None else None)
    n = q.shape[0] + 2 * max(q.shape[-1], v.shape[-1]) + 24
    f = 2.0 ** -24
    b = {}
    for name, size in sizes.items():
        fp32_result = name in ("state", "dstate0")
        inner = (0.0 if fp32_result or u == f else u) + n * f
        b[name] = (f if fp32_result else u) * want[name].abs() + inner * size + 1e-30
    if dout is not None:
        # the pairs' sums of a chunk cancel in dg: each is a sum over (a part of) all tokens from t on
        qdq, kdk = (q.double().abs() * sizes["dq"]).sum(-1), (k.double().abs() * sizes["dk"]).sum(-1)
        b["dg"] = U[g.dtype] * want["dg"].abs() + (0.0 if u == f else 2 * u) * sizes["dg"] + n * f * (sizes["dg"] + (qdq + kdk).flip(0).cumsum(0).flip(0)) + 1e-30
    return b


def norm(x, w, residual=None, eps=1e-6, dy=None, dh=None):
    h = (x.double() + residual.double()).to(x.dtype) if residual is not None else x
    hd, wd = h.double(), w.double()
    r = 1 / (hd.square().mean(-1, keepdim=True) + eps).sqrt()
    got = {"h": h, "y": hd * r * wd, "rstd": r}
    if dy is not None:
        n, d = hd * r, dy.double()
        got["dx"] = r * (d * wd - n * (d * wd * n).mean(-1, keepdim=True)) + (dh.double() if dh is not None else 0.0)
        got["dw"] = (d * n).flatten(0, -2).sum(0)
        got["dx_size"] = r * ((d * wd).abs() + n.abs() * (d * wd * n).abs().mean(-1, keepdim=True)) + (dh.double().abs() if dh is not None else 0.0)
        got["dw_size"] = (d * n).abs().flatten(0, -2).sum(0)
    return got
