"""Timed cases of the sequence operators beside the GRU: linear attention with a decay for each head, over whole sequences
(``attention``), with its gradient (``train``) and for single tokens (``step``), and the root-mean-square norm with the
residual's addition, with its gradient (``norm_train``) and with 8-bit output (``norm_q8``).

A case is a dict.  Attention: ``T``, ``B``, ``H`` (heads), ``Hk`` (heads of q and k, each shared by H / Hk heads), ``Dk``,
``Dv``, ``dtype``, ``h0`` (an initial state is passed), ``ragged`` (sequences of different lengths), ``batch_first``,
``fused`` (q, k and v are parts of one projection's output, as a layer has them).  Norm: ``rows``, ``cols``, ``dtype``,
``residual``.

The plain form of the attention is the definition written out over all pairs of tokens, in 32 bits with the decays' running
sums in 64; ``exact`` is the recurrence token by token in 64 bits.
"""
import importlib
import math

import torch

own = False

_TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}
_DEFAULTS = {"Hk": 0, "h0": False, "ragged": False, "batch_first": False, "fused": False, "residual": True, "dtype": "bfloat16"}
_EPS = 1e-6


def _case(**kw):
    return {**_DEFAULTS, **kw}


def listed():
    return [
        # a short phrase continued from a carried state: call latency
        _case(name="att_phrase", do="attention", T=24, B=1, H=4, Dk=64, Dv=64, h0=True, fused=True),
        # a batch of long sequences through a layer 1024 wide
        _case(name="att_batch", do="attention", T=1000, B=64, H=16, Dk=64, Dv=64, fused=True),
        # one recording, very long, wide heads: little to run side by side but time itself
        _case(name="att_long", do="attention", T=16000, B=1, H=4, Dk=128, Dv=128, h0=True),
        # sizes that are no multiple of anything, padded batch, fp32
        _case(name="att_ragged_odd", do="attention", T=127, B=37, H=5, Dk=40, Dv=72, ragged=True, dtype="float32", batch_first=True),
        # training step of a wide layer in bf16
        _case(name="train_bf16", do="train", T=1000, B=16, H=8, Dk=128, Dv=128, fused=True),
        # fp32 training of a padded batch from given states, keys shared by two heads
        _case(name="train_fp32_ragged", do="train", T=200, B=32, H=8, Hk=4, Dk=64, Dv=64, ragged=True, h0=True, dtype="float32"),
        # one frame of a stream
        _case(name="step_one", do="step", B=1, H=4, Dk=64, Dv=64),
        # a token for each of many streams
        _case(name="step_batch", do="step", B=256, H=16, Dk=128, Dv=128),
        # one frame's norm before a quantized layer
        _case(name="norm_q8_row", do="norm_q8", rows=1, cols=512),
        # the bidirectional encoder's output (512 units each way), 256 sequences of 200 steps
        _case(name="norm_q8_encoder", do="norm_q8", rows=51200, cols=1024),
        # training of the same
        _case(name="norm_train_encoder", do="norm_train", rows=51200, cols=1024),
        # odd width, fp32
        _case(name="norm_train_odd", do="norm_train", rows=4699, cols=321, dtype="float32", residual=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    do = rng.choices(["attention", "train", "step", "norm_q8", "norm_train"], [4, 3, 2, 2, 2])[0]
    dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
    if do.startswith("norm"):
        while True:
            c = _case(do=do, rows=_log(rng, 1, 60000), cols=_log(rng, 16, 8192), dtype=dtype, residual=rng.random() < 0.7)
            if c["rows"] * c["cols"] * (2 if dtype == "float32" else 1) <= 51200 * 1024:
                return c

    def size():
        return rng.choice([64, 64, 128, 128, 32, 96, 8 * rng.randint(2, 16), rng.randint(5, 128)])

    while True:
        c = _case(do=do, T=1 if do == "step" else _log(rng, 1, 16000 if do == "attention" else 4000), B=_log(rng, 1, 256),
                  H=_log(rng, 1, 16), Dk=size(), Dv=size(), dtype=dtype, h0=rng.random() < 0.4 and do != "step",
                  ragged=rng.random() < 0.4 and do != "step", batch_first=rng.random() < 0.4, fused=rng.random() < 0.5)
        share = rng.choice([1, 1, 1, 2, 4])
        c["Hk"] = c["H"] // share if c["H"] % share == 0 else 0
        T, rows = c["T"], c["B"] * c["H"]
        if do == "step":
            if rows * c["Dk"] * c["Dv"] <= 256 * 16 * 128 * 128 and rows >= 2:
                return c
        elif rows * T * T <= 1.0e9 and rows * T * max(c["Dk"], c["Dv"]) <= (6.5e7 if do == "attention" else 1.6e7):
            return c


# ------------------------------------------------------------------------------------- inputs
def _dims(c):
    return c["B"], c["H"], c["Hk"] or c["H"], c["Dk"], c["Dv"]


def prepare(case, seed):
    c = {**_DEFAULTS, **case}
    dev, dt = torch.device("cuda", torch.cuda.current_device()), _TYPES[c["dtype"]]
    gen = torch.Generator(device=dev).manual_seed(int(seed) % (1 << 60))

    def randn(*shape, sigma=1.0, dtype=dt):
        return (torch.randn(shape, generator=gen, device=dev) * sigma).to(dtype)

    s = {"case": c}
    if c["do"].startswith("norm"):
        n, d = c["rows"], c["cols"]
        s["x"] = randn(n, d)
        # the stream has grown over the layers and has a few loud columns
        s["r"] = (randn(n, d, sigma=2.0, dtype=torch.float32) * (1 + 6 * (torch.rand(d, generator=gen, device=dev) < 0.01))).to(dt) if c["residual"] else None
        s["w"] = (1 + 0.2 * torch.randn(d, generator=gen, device=dev)).to(dt)
        if c["do"] == "norm_train":
            s["dy"], s["dh"] = randn(n, d), randn(n, d)
        return s
    B, H, Hk, Dk, Dv = _dims(c)
    lead = (B,) if c["do"] == "step" else (B, c["T"]) if c["batch_first"] else (c["T"], B)
    if c["fused"]:
        qkv = randn(*lead, 2 * Hk * Dk + H * Dv)
        q, k, v = qkv.split([Hk * Dk, Hk * Dk, H * Dv], dim=-1)
        s["q"], s["k"], s["v"] = q.unflatten(-1, (Hk, Dk)), k.unflatten(-1, (Hk, Dk)), v.unflatten(-1, (H, Dv))
    else:
        s["q"], s["k"], s["v"] = randn(*lead, Hk, Dk), randn(*lead, Hk, Dk), randn(*lead, H, Dv)
    # a gate per token and head, whose bias gives the heads memories from a few tokens to a thousand
    bias = torch.linspace(1.0, 7.0, H, device=dev)
    s["g"] = -torch.nn.functional.softplus(torch.randn((*lead, H), generator=gen, device=dev) - bias).to(dt)
    if c["do"] == "step":
        s["state"] = randn(B, H, Dk, Dv, dtype=torch.float32)
        return s
    s["state"] = randn(B, H, Dk, Dv, dtype=torch.float32) if c["h0"] else None
    s["lengths"] = None
    if c["ragged"]:
        n = torch.randint(0, c["T"] + 1, (B,), generator=gen, device=dev, dtype=torch.int32)
        n[int(torch.randint(0, B, (1,), generator=gen, device=dev))] = c["T"]
        s["lengths"] = n
    if c["do"] == "train":
        s["dout"] = randn(*lead, H, Dv)
        s["dstate"] = randn(B, H, Dk, Dv, dtype=torch.float32)
    return s


# --------------------------------------------------------------------------------- plain forms
def _heads(c, x, H, kind):
    """[T, B, heads, D] (or [B, T, ...]) -> [B, H, T, D] of `kind`."""
    x = x.to(kind)
    if not c["batch_first"]:
        x = x.transpose(0, 1)
    x = x.transpose(1, 2)
    return x.repeat_interleave(H // x.shape[1], dim=1) if x.shape[1] != H else x


def _back(c, x, heads=None):
    """The other way, with the sum over heads that share one."""
    if heads is not None and heads != x.shape[1]:
        x = x.unflatten(1, (heads, -1)).sum(2)
    x = x.transpose(1, 2)
    return (x if c["batch_first"] else x.transpose(0, 1)).contiguous()


def _plain_attention(s):
    c = s["case"]
    B, H, Hk, Dk, Dv = _dims(c)
    T, scale, dt = c["T"], c["Dk"] ** -0.5, s["q"].dtype
    f = torch.float32
    q, k, v = _heads(c, s["q"], H, f), _heads(c, s["k"], H, f), _heads(c, s["v"], H, f)
    g = _heads(c, s["g"].unsqueeze(-1), H, torch.float64).squeeze(-1)
    valid = None
    if s["lengths"] is not None:
        valid = (torch.arange(T, device=q.device) < s["lengths"][:, None])[:, None, :]
        q, k, v = (torch.where(valid[..., None], x, 0.0) for x in (q, k, v))
        g = torch.where(valid, g, 0.0)
    G = g.cumsum(-1)
    D = (G[..., :, None] - G[..., None, :]).float()
    D.masked_fill_(torch.ones(T, T, dtype=torch.bool, device=q.device).triu_(1), -math.inf).exp_()
    D.mul_(scale)
    from_start, to_end, whole = G.exp().float(), (G[..., -1:] - G).exp().float(), G[..., -1].exp().float()
    A = q @ k.transpose(-1, -2)
    o = (A * D) @ v
    state = (k * to_end[..., None]).transpose(-1, -2) @ v
    if s["state"] is not None:
        inter = (q * (scale * from_start)[..., None]) @ s["state"]
        o = o + inter
        state = state + whole[..., None, None] * s["state"]
    got = {"out": _back(c, o).to(dt), "state": state}
    if c["do"] == "attention":
        return got
    do = _heads(c, s["dout"], H, f)
    if valid is not None:
        do = torch.where(valid[..., None], do, 0.0)
    dst = s["dstate"]
    E = do @ v.transpose(-1, -2)
    W = (A * E * D).double()                                   # each pair's part of the loss's change with its decay
    dG = W.sum(-1) - W.sum(-2)
    E *= D
    kd, vd = k * to_end[..., None], v * to_end[..., None]
    dk_end = vd @ dst.transpose(-1, -2)
    dq, dk, dv = E @ k, E.transpose(-1, -2) @ q + dk_end, (A * D).transpose(-1, -2) @ do + kd @ dst
    dG -= (dk_end * k).double().sum(-1)
    if s["state"] is not None:
        dq += scale * from_start[..., None] * (do @ s["state"].transpose(-1, -2))
        dG += (inter * do).double().sum(-1)
        got["dstate0"] = whole[..., None, None] * dst + (q * (scale * from_start)[..., None]).transpose(-1, -2) @ do
    dG[..., -1] += (state.double() * dst).sum((-1, -2))
    dg = dG.flip(-1).cumsum(-1).flip(-1)
    if valid is not None:
        dg = torch.where(valid, dg, 0.0)
    got.update(dq=_back(c, dq, Hk).to(dt), dk=_back(c, dk, Hk).to(dt), dv=_back(c, dv).to(dt), dg=_back(c, dg[..., None]).squeeze(-1).to(dt))
    return got


def _plain_step(s):
    c = s["case"]
    B, H, Hk, Dk, Dv = _dims(c)
    q, k, v, g = (s[n].float() for n in ("q", "k", "v", "g"))
    q, k = q.repeat_interleave(H // Hk, 1), k.repeat_interleave(H // Hk, 1)
    state = s["state"].mul_(g.exp()[..., None, None]).add_(k[..., :, None] * v[..., None, :])      # carried on in place
    out = (q[..., None, :] @ state).squeeze(-2) * Dk ** -0.5
    return {"out": out.to(s["q"].dtype), "state": state}


def _plain_norm(s):
    c, dt = s["case"], s["x"].dtype
    h = (s["x"].float() + s["r"].float()).to(dt) if s["r"] is not None else s["x"]
    hf, w = h.float(), s["w"].float()
    r = (hf.square().mean(-1, keepdim=True) + _EPS).rsqrt()
    got = {"h": h} if s["r"] is not None else {}
    if c["do"] == "norm_q8":
        # next to a border of the rounding 32 bits decide wrongly; the row's root mean square is no part of the ratio
        hw = h.double() * s["w"].double()
        m = hw.abs().amax(-1, keepdim=True)
        q = torch.where(m > 0, torch.round(hw * 127 / m), 0.0)
        scale = (m.float() * r / 127)
        return {**got, "y": (q.float() * scale).to(dt), "scale": scale.squeeze(-1)}
    got["y"] = (hf * r * w).to(dt)
    dyw, dy = s["dy"].float() * w, s["dy"].float()
    n = hf * r
    dx = r * (dyw - n * (dyw * n).mean(-1, keepdim=True))
    if s["r"] is not None:
        dx = dx + s["dh"].float()
    got["dx"] = dx.to(dt)
    got["dw"] = (dy * n).sum(0).to(dt)
    return got


# ------------------------------------------------------------------------- the framework's calls
def _package(name):
    entry = importlib.import_module("__graft_entry__")
    entry.load_package()
    return importlib.import_module(f"{entry.PKG_NAME}.{name}")


def _own_attention(s):
    c, la = s["case"], _package("linear_attention")
    if c["do"] == "attention":
        out, state = la.linear_attention(s["q"], s["k"], s["v"], s["g"], s["state"], lengths=s["lengths"], batch_first=c["batch_first"])
        return {"out": out, "state": state}
    names = ["q", "k", "v", "g"] + (["state"] if s["state"] is not None else [])
    leaves = [s[n].detach().requires_grad_() for n in names]
    out, state = la.linear_attention(*leaves, lengths=s["lengths"], batch_first=c["batch_first"])
    grads = torch.autograd.grad((out, state), leaves, (s["dout"], s["dstate"]))
    got = dict(zip(["dq", "dk", "dv", "dg", "dstate0"], grads))
    return {"out": out.detach(), "state": state.detach(), **got}


def _own_step(s):
    la = _package("linear_attention")
    out = la.linear_attention_step(s["q"], s["k"], s["v"], s["g"], s["state"])
    return {"out": out, "state": s["state"]}


def _own_norm(s):
    c, norm = s["case"], _package("norm")
    if c["do"] == "norm_q8":
        q, scale, *h = norm.rms_norm_q8(s["x"], s["w"], residual=s["r"], eps=_EPS)
        got = {"y": torch.mul(q, scale.unsqueeze(-1), out=torch.empty_like(s["x"])), "scale": scale}
        return {**got, "h": h[0]} if h else got
    x, w = s["x"].detach().requires_grad_(), s["w"].detach().requires_grad_()
    if s["r"] is None:
        y = norm.rms_norm(x, w, eps=_EPS)
        dx, dw = torch.autograd.grad(y, (x, w), s["dy"])
        return {"y": y.detach(), "dx": dx, "dw": dw}
    y, h = norm.rms_norm(x, w, residual=s["r"], eps=_EPS)
    dx, dw = torch.autograd.grad((y, h), (x, w), (s["dy"], s["dh"]))
    return {"y": y.detach(), "h": h.detach(), "dx": dx, "dw": dw}


def run(state):
    do = state["case"]["do"]
    if do in ("attention", "train"):
        return _own_attention(state) if own else _plain_attention(state)
    if do == "step":
        return _own_step(state) if own else _plain_step(state)
    return _own_norm(state) if own else _plain_norm(state)


# ------------------------------------------------------------------------------------- 64 bits
def _exact_attention(s):
    """The recurrence, one token after the other, and its adjoint."""
    c = s["case"]
    B, H, Hk, Dk, Dv = _dims(c)
    T, f = c["T"], torch.float64
    if c["do"] == "train" and T * B * H * Dk * Dv * 8 > 50e9:
        return None
    time_first = (lambda x: x.transpose(0, 1)) if c["batch_first"] else (lambda x: x)
    q, k, v, g = (time_first(s[n]).to(f) for n in ("q", "k", "v", "g"))
    q, k = (x.repeat_interleave(H // Hk, 2) for x in (q, k))
    on = torch.ones(T, B, dtype=torch.bool, device=q.device)
    if s["lengths"] is not None:
        on = torch.arange(T, device=q.device)[:, None] < s["lengths"][None, :]
    a = torch.where(on[..., None], g.exp(), 1.0)
    w = on.to(f)[..., None, None] / math.sqrt(Dk)
    k = k * on[..., None, None]
    S = s["state"].to(f) if s["state"] is not None else torch.zeros(B, H, Dk, Dv, dtype=f, device=q.device)
    train, states, outs = c["do"] == "train", [S], []
    for t in range(T):
        S = torch.addcmul(k[t, :, :, :, None] * v[t, :, :, None, :], a[t, :, :, None, None], S)
        outs.append(torch.einsum("bhk,bhkv->bhv", q[t], S))
        if train:
            states.append(S)
    got = {"out": time_first(torch.stack(outs) * w), "state": S}
    if train:
        do, dS = time_first(s["dout"]).to(f) * w, s["dstate"].to(f)
        dq, dk, dv, dg = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v), torch.empty_like(g)
        for t in reversed(range(T)):
            dS = dS + q[t, :, :, :, None] * do[t, :, :, None, :]
            dq[t] = torch.einsum("bhkv,bhv->bhk", states[t + 1], do[t])
            dk[t] = torch.einsum("bhkv,bhv->bhk", dS, v[t])
            dv[t] = torch.einsum("bhkv,bhk->bhv", dS, k[t])
            dg[t] = (dS * states[t]).sum((-1, -2)) * a[t]
            dS = dS * a[t, :, :, None, None]
        on = on[..., None]
        dk, dg = dk * on[..., None], dg * on
        got.update(dq=time_first(dq.unflatten(2, (Hk, -1)).sum(3)), dk=time_first(dk.unflatten(2, (Hk, -1)).sum(3)), dv=time_first(dv), dg=time_first(dg))
        if s["state"] is not None:
            got["dstate0"] = dS
    return got


def exact(case, seed):
    s = prepare(case, seed)
    c, f = s["case"], torch.float64
    if c["do"] in ("attention", "train"):
        return _exact_attention(s)
    if c["do"] == "step":
        group = c["H"] // (c["Hk"] or c["H"])
        q, k = (s[n].to(f).repeat_interleave(group, 1) for n in ("q", "k"))
        S = torch.einsum("bhk,bhv->bhkv", k, s["v"].to(f)) + s["g"].to(f).exp()[..., None, None] * s["state"].to(f)
        return {"out": torch.einsum("bhk,bhkv->bhv", q, S) / math.sqrt(c["Dk"]), "state": S}
    h, w, got = s["x"].to(f), s["w"].to(f), {}
    if s["r"] is not None:
        h = got["h"] = h + s["r"].to(f)
        h = h.to(s["x"].dtype).to(f)          # the stream is what the next layer reads
    y = h * w / torch.sqrt((h * h).mean(1, keepdim=True) + _EPS)
    if c["do"] == "norm_q8":
        scale = y.abs().amax(1) / 127
        return {**got, "y": torch.round(y / scale.clamp_min(1e-300)[:, None]) * scale[:, None], "scale": scale}
    h = h.requires_grad_()
    w = w.requires_grad_()
    y = h * w / torch.sqrt((h * h).mean(1, keepdim=True) + _EPS)
    dx, dw = torch.autograd.grad(y, (h, w), s["dy"].to(f))
    return {**got, "y": y.detach(), "dx": dx + s["dh"].to(f) if s["r"] is not None else dx, "dw": dw}


def work(case):
    """Each input read once and each output written once; the operations of the recurrence, which are the fewest."""
    c = {**_DEFAULTS, **case}
    e = 4 if c["dtype"] == "float32" else 2
    if c["do"].startswith("norm"):
        n, d = c["rows"], c["cols"]
        tensors = 1 + 2 * c["residual"]                              # x; residual read, stream written
        if c["do"] == "norm_q8":
            return {"bytes": n * d * (tensors * e + 1) + d * e + 4 * n, "flops": 6 * n * d}
        return {"bytes": n * d * e * (tensors + 1 + 2 + 2 * c["residual"]) + 2 * d * e, "flops": 14 * n * d}
    B, H, Hk, Dk, Dv = _dims(c)
    n, states = B * (1 if c["do"] == "step" else c["T"]), 4 * B * H * Dk * Dv
    read = 2 * Hk * Dk + H * Dv + H
    if c["do"] == "train":                                           # q, k, v, g, dout and their gradients, out
        return {"bytes": n * e * (2 * read + 2 * H * Dv) + states * (2 + 2 * c["h0"]), "flops": 14 * n * H * Dk * Dv}
    return {"bytes": n * e * (read + H * Dv) + states * (1 + (c["h0"] or c["do"] == "step")), "flops": 5 * n * H * Dk * Dv}
