"""Linear attention with a decay for each head against the recurrence in 64 bits, token by token (tests/seq_reference.py, which
also says how far a result may be off)."""
import importlib

import pytest
import torch

from __graft_entry__ import PKG_NAME
from tests import seq_reference as ref

la = importlib.import_module(PKG_NAME + ".linear_attention")
pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def make(dev, T, B, H, Dk, Dv, dtype, Hk=None, seed=0, h0=True, lengths=None, decay=F32, memory=(1.0, 7.0), batch_first=False, fused=False):
    gen = torch.Generator(device=dev).manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=gen, device=dev)

    Hk = Hk or H
    lead = (B, T) if batch_first else (T, B)
    if fused:          # parts of one projection's output
        qkv = randn(*lead, 2 * Hk * Dk + H * Dv).to(dtype)
        q, k, v = (x.unflatten(-1, (h, -1)) for x, h in zip(qkv.split([Hk * Dk, Hk * Dk, H * Dv], -1), (Hk, Hk, H)))
    else:
        q, k, v = randn(*lead, Hk, Dk).to(dtype), randn(*lead, Hk, Dk).to(dtype), randn(*lead, H, Dv).to(dtype)
    g = -torch.nn.functional.softplus(randn(*lead, H) - torch.linspace(*memory, H, device=dev)).to(decay)
    state = randn(B, H, Dk, Dv) if h0 else None
    n = torch.tensor(lengths, dtype=torch.int32, device=dev) if lengths is not None else None
    return q, k, v, g, state, n


def want_of(q, k, v, g, state, n, batch_first=False, scale=None, dout=None, dstate=None):
    """64-bit results and bounds, in the layout of the arguments; gradients of shared heads summed."""
    t = (lambda x: x.transpose(0, 1)) if batch_first else (lambda x: x)
    H, Hk = v.shape[2], q.shape[2]
    args = [t(x).repeat_interleave(H // Hk, 2) for x in (q, k)] + [t(v), t(g.expand(*v.shape[:3]))]
    kw = dict(state=state, lengths=n, scale=scale, dout=t(dout) if dout is not None else None, dstate=dstate)
    want = ref.attention(*args, **kw)
    bound = ref.attention_bounds(want, *args, **kw)
    for r in (want, bound):
        for name in ("dq", "dk"):
            if name in r:
                r[name] = r[name].unflatten(2, (Hk, -1)).sum(3)
        for name in ("out", "dq", "dk", "dv", "dg"):
            if name in r:
                r[name] = t(r[name])
    return want, bound


def hold(got, want, bound):
    for name, x in got.items():
        assert torch.isfinite(x).all(), name
        off = (x.double() - want[name]).abs() / bound[name]
        assert off.max() <= 1, f"{name}: {off.max():.2f} times the bound, at {[int(i) for i in (off == off.max()).nonzero()[0]]}"


SHAPES = [  # T, B, H, Dk, Dv
    (1, 1, 1, 1, 1), (1, 3, 2, 64, 64), (24, 1, 4, 64, 64), (63, 2, 3, 64, 64), (64, 2, 2, 64, 128), (65, 2, 2, 128, 64), (127, 3, 5, 40, 72),
    (128, 2, 2, 128, 128), (129, 1, 2, 128, 128), (300, 2, 2, 33, 17), (257, 1, 3, 96, 8), (200, 2, 2, 200, 256), (700, 1, 2, 64, 64), (1500, 1, 1, 128, 128),
]


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward(shape, dtype, cuda_device):
    q, k, v, g, state, n = make(cuda_device, *shape, dtype)
    want, bound = want_of(q, k, v, g, state, n)
    out, last = la.linear_attention(q, k, v, g, state)
    assert out.dtype == dtype and last.dtype == F32
    hold({"out": out, "state": last}, want, bound)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_gradients(shape, dtype, cuda_device):
    q, k, v, g, state, n = make(cuda_device, *shape, dtype, decay=dtype)
    leaves = [t.requires_grad_() for t in (q, k, v, g, state)]
    out, last = la.linear_attention(*leaves)
    dout, dstate = torch.randn_like(out), torch.randn_like(last)
    grads = torch.autograd.grad((out, last), leaves, (dout, dstate))
    want, bound = want_of(*[t.detach() for t in leaves], None, dout=dout, dstate=dstate)
    hold(dict(zip(("dq", "dk", "dv", "dg", "dstate0"), grads)), want, bound)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("case", [
    dict(T=150, B=5, H=4, Dk=64, Dv=64, Hk=2, lengths=[0, 1, 128, 150, 77], fused=True),
    dict(T=150, B=4, H=4, Dk=64, Dv=64, Hk=1, lengths=[150, 64, 65, 900], batch_first=True),
    dict(T=260, B=3, H=2, Dk=128, Dv=128, lengths=[-5, 260, 129], batch_first=True, fused=True),
    dict(T=131, B=2, H=6, Dk=24, Dv=40, Hk=3, lengths=[131, 2], h0=False),
    dict(T=131, B=2, H=6, Dk=23, Dv=41, Hk=3, h0=False, fused=True),
], ids=lambda c: "-".join(f"{k}{v}" for k, v in c.items()))
def test_padded_batches_shared_heads_and_strides(case, dtype, cuda_device):
    q, k, v, g, state, n = make(cuda_device, dtype=dtype, decay=dtype, **case)
    bf = case.get("batch_first", False)
    leaves = [t.detach().requires_grad_() for t in (q, k, v, g)] + ([state.requires_grad_()] if state is not None else [])
    out, last = la.linear_attention(*leaves, lengths=n, batch_first=bf)
    dout, dstate = torch.randn_like(out), torch.randn_like(last)
    grads = torch.autograd.grad((out, last), leaves, (dout, dstate))
    want, bound = want_of(q, k, v, g, state.detach() if state is not None else None, n, bf, dout=dout, dstate=dstate)
    hold({"out": out, "state": last, **dict(zip(("dq", "dk", "dv", "dg", "dstate0"), grads))}, want, bound)
    if n is not None:      # behind the sequences: zeros
        T = case["T"]
        past = torch.arange(T, device=cuda_device)[:, None] >= n[None, :]
        for x in (out, *grads[:4]):
            x = x.transpose(0, 1) if bf else x
            assert (x[past] == 0).all()


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_what_lies_behind_a_sequence_is_not_read(dtype, cuda_device):
    q, k, v, g, state, n = make(cuda_device, 200, 3, 2, 64, 64, dtype, lengths=[100, 0, 200])
    clean = [t.clone() for t in (q, k, v, g)]
    past = torch.arange(200, device=cuda_device)[:, None] >= n[None, :]
    for t in (q, k, v, g):
        t[past] = float("nan")
    v[past] = float("inf")
    dout = torch.randn(200, 3, 2, 64, device=cuda_device).to(dtype)
    got, ref_ = [], []
    for to, args in ((got, (q, k, v, g)), (ref_, clean)):
        leaves = [t.requires_grad_() for t in args]
        out, last = la.linear_attention(*leaves, initial_state=state, lengths=n)
        to += [out.detach(), last.detach(), *torch.autograd.grad(out, leaves, torch.where(past[..., None, None], float("nan"), dout) if to is got else dout)]
    assert all(torch.equal(a, b) for a, b in zip(got, ref_))
    assert torch.equal(got[1][1], state[1])


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("D", [64, 128])
def test_later_tokens_do_not_reach_earlier_outputs(D, dtype, cuda_device):
    q, k, v, g, state, _ = make(cuda_device, 300, 2, 2, D, D, dtype)
    first = la.linear_attention(q, k, v, g, state)[0]
    for t in (q, k, v, g):
        t[150, 0] = float("nan")
    v[151:, 0] = float("inf")
    out = la.linear_attention(q, k, v, g, state)[0]
    # the sums of a chunk with such a token may be taken in another order than those of a clean one
    want, bound = want_of(q[:150], k[:150], v[:150], g[:150], state, None)
    hold({"out": out[:150]}, want, bound)
    assert torch.isnan(out[150:, 0]).all() and torch.equal(out[:, 1], first[:, 1])


def test_decays_of_nothing_and_of_everything(cuda_device):
    q, k, v, g, state, _ = make(cuda_device, 200, 2, 2, 64, 64, F32)
    g[:] = 0.0
    g[70] = float("-inf")                   # starts anew
    g[100:140] = -300.0                     # each of them is nothing in fp32
    want, bound = want_of(q, k, v, g, state, None)
    out, last = la.linear_attention(q, k, v, g, state)
    hold({"out": out, "state": last}, want, bound)
    fresh = la.linear_attention(q[70:], k[70:], v[70:], g[70:])[0]
    hold({"out": fresh}, {"out": want["out"][70:]}, {"out": bound["out"][70:]})


@pytest.mark.parametrize("decay", [F32, BF], ids=["fp32", "bf16"])
def test_constant_decays_and_scale(decay, cuda_device):
    q, k, v, _, state, _ = make(cuda_device, 140, 2, 3, 64, 64, BF)
    g = torch.tensor([-0.5, -0.01, -0.001], device=cuda_device).to(decay).requires_grad_()
    out, last = la.linear_attention(q, k, v, g, state, scale=-0.3)
    want, bound = want_of(q, k, v, g.detach(), state, None, scale=-0.3, dout=torch.ones_like(out))
    hold({"out": out.detach(), "state": last.detach()}, want, bound)
    dg, = torch.autograd.grad(out, g, torch.ones_like(out))
    assert dg.shape == (3,)
    per_token = bound["dg"] + (0 if decay == BF else 2.0 ** -24) * want["dg"].abs()
    off = (dg.double() - want["dg"].sum((0, 1))).abs()
    assert (off <= per_token.sum((0, 1)) + ref.U[decay] * want["dg"].sum((0, 1)).abs() + 2.0 ** -24 * 280 * want["dg"].abs().sum((0, 1))).all()


def test_gradients_against_differences(cuda_device):
    """d loss along a direction, by the gradients and by two forwards in fp32."""
    q, k, v, g, state, n = make(cuda_device, 100, 2, 2, 48, 56, F32, lengths=[100, 33], memory=(1.0, 3.0))
    leaves = [t.requires_grad_() for t in (q, k, v, g, state)]
    out, last = la.linear_attention(*leaves, lengths=n)
    a, b = torch.randn_like(out), torch.randn_like(last)
    grads = torch.autograd.grad((out, last), leaves, (a, b))
    for i in range(5):
        d = torch.randn_like(leaves[i])
        eps = 1e-2 / d.abs().max()
        with torch.no_grad():
            s = []
            for e in (eps, -eps):
                x = [t + e * d if j == i else t for j, t in enumerate(leaves)]
                o, l = la.linear_attention(*x, lengths=n)
                s.append((o.double() * a).sum() + (l.double() * b).sum())
        along = (s[0] - s[1]) / (2 * eps.double())
        # third derivatives: only the decays' (exp), 1/6 eps^2 relative; fp32: sums of about 1e4 terms of size 1, 2^-24 each, over 2 eps
        tol = 1e-3 * grads[i].double().norm() * d.double().norm() * 1e-1 + 1e4 ** 0.5 * 2.0 ** -24 * 10 * (a.norm() + b.norm()).double() / (2 * eps)
        assert abs(along - (grads[i].double() * d).sum()) <= tol


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("B,H,Hk,Dk,Dv", [(1, 1, 1, 1, 1), (1, 4, 4, 64, 64), (3, 6, 2, 40, 72), (2, 2, 2, 128, 128), (5, 3, 3, 33, 17), (2, 2, 1, 200, 256), (1, 2, 2, 256, 255), (300, 16, 16, 64, 64)])
def test_step(B, H, Hk, Dk, Dv, dtype, cuda_device):
    q, k, v, g, state, _ = make(cuda_device, 1, B, H, Dk, Dv, dtype, Hk=Hk)
    want, bound = want_of(q, k, v, g, state, None)
    out = la.linear_attention_step(q[0], k[0], v[0], g[0], state)
    hold({"out": out[None], "state": state}, want, bound)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_steps_continue_a_prompt(dtype, cuda_device):
    q, k, v, g, state, _ = make(cuda_device, 140, 2, 4, 64, 64, dtype, Hk=2, fused=True)
    want, bound = want_of(q, k, v, g, state, None)
    version = state._version
    out, last = la.linear_attention(q[:130], k[:130], v[:130], g[:130], state)
    assert state._version == version
    outs = [out] + [la.linear_attention_step(q[t], k[t], v[t], g[t], last)[None] for t in range(130, 140)]
    assert last._version == 10
    hold({"out": torch.cat(outs), "state": last}, want, bound)


def test_step_on_parts_of_a_pool_of_states(cuda_device):
    q, k, v, g, _, _ = make(cuda_device, 1, 4, 3, 64, 64, F32)
    pool = torch.randn(9, 5, 64, 64, device=cuda_device)
    before, part = pool.clone(), pool[1::2, 1:4]
    want, bound = want_of(q, k, v, g, part.clone(), None)
    out = la.linear_attention_step(q[0], k[0], v[0], g[0], part)
    hold({"out": out[None], "state": part}, want, bound)
    rest = torch.ones(9, 5, dtype=torch.bool)
    rest[1::2, 1:4] = False
    assert torch.equal(pool[rest], before[rest])
    flipped = torch.randn(3, 4, 64, 64, device=cuda_device).transpose(0, 1)      # heads outside
    want, bound = want_of(q, k, v, g, flipped.clone(), None)
    out = la.linear_attention_step(q[0], k[0], v[0], g[0], flipped)
    hold({"out": out[None], "state": flipped}, want, bound)


def test_nothing_to_do(cuda_device):
    for T, B in ((0, 2), (5, 0), (0, 0)):
        q, k, v, g, state, _ = make(cuda_device, T, B, 2, 64, 32, BF)
        leaves = [t.requires_grad_() for t in (q, k, v, g, state)]
        out, last = la.linear_attention(*leaves)
        assert out.shape == (T, B, 2, 32) and torch.equal(last, state)
        grads = torch.autograd.grad((out, last), leaves, (torch.ones_like(out), torch.full_like(last, 2.0)))
        assert [x.shape for x in grads] == [x.shape for x in leaves] and (grads[4] == 2).all()
    q, k, v, g, _, _ = make(cuda_device, 1, 0, 2, 64, 32, BF)
    assert la.linear_attention_step(q[0], k[0], v[0], g[0], torch.empty(0, 2, 64, 32, device=cuda_device)).shape == (0, 2, 32)


def test_only_some_gradients(cuda_device):
    q, k, v, g, state, _ = make(cuda_device, 70, 2, 2, 64, 64, F32)
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v, g, state)]
    out, last = la.linear_attention(*leaves)
    all_ = torch.autograd.grad(last.sum(), leaves)                # nothing comes from out
    v1 = v.detach().clone().requires_grad_()
    out, last = la.linear_attention(q, k, v1, g, state)
    last.sum().backward()
    assert torch.equal(v1.grad, all_[2])


def test_same_results_every_time_and_on_other_streams(cuda_device):
    q, k, v, g, state, _ = make(cuda_device, 900, 2, 4, 64, 64, BF, decay=BF)
    leaves = [t.requires_grad_() for t in (q, k, v, g, state)]

    def run():
        out, last = la.linear_attention(*leaves)
        return [out.detach(), last.detach(), *torch.autograd.grad((out, last), leaves, (torch.ones_like(out), torch.ones_like(last)))]

    first = run()
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(run())
    torch.cuda.synchronize()
    for r in got:
        assert all(torch.equal(a, b) for a, b in zip(first, r))


def test_two_captured_graphs(cuda_device):
    """A prompt and a step, and another prompt, captured and replayed in turn with new inputs."""
    sets = [make(cuda_device, 300, 2, 4, 64, 64, BF, seed=s) for s in (1, 2)]
    graphs, outs = [], []
    with torch.no_grad():
        for q, k, v, g, state, _ in sets:
            la.linear_attention(q, k, v, g, state)
        torch.cuda.synchronize()
        for q, k, v, g, state, _ in sets:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                o, last = la.linear_attention(q, k, v, g, state)
                s = la.linear_attention_step(q[0], k[0], v[0], g[0], last)
            graphs.append(graph)
            outs.append((o, last, s))
        for again in range(2):
            for q, *_ in sets:
                q.mul_(-1.0)
            for graph in graphs:
                graph.replay()
            torch.cuda.synchronize()
            for (q, k, v, g, state, _), got in zip(sets, outs):
                o, last = la.linear_attention(q, k, v, g, state)
                s = la.linear_attention_step(q[0], k[0], v[0], g[0], last)
                assert torch.equal(o, got[0]) and torch.equal(last, got[1]) and torch.equal(s, got[2])


def test_saved_tensors_may_move(cuda_device):
    q, k, v, g, state, _ = make(cuda_device, 150, 2, 2, 64, 64, BF, decay=BF)
    leaves = [t.requires_grad_() for t in (q, k, v, g, state)]
    want = torch.autograd.grad(la.linear_attention(*leaves)[0].float().square().sum(), leaves)

    def odd(t):          # a copy off its alignment
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:]
        flat.copy_(t.reshape(-1))
        return flat.view(t.shape)

    with torch.autograd.graph.saved_tensors_hooks(odd, lambda t: t):
        out = la.linear_attention(*leaves)[0]
    got = torch.autograd.grad(out.float().square().sum(), leaves)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.to(cuda_device)):
        out = la.linear_attention(*leaves)[0]
    got = torch.autograd.grad(out.float().square().sum(), leaves)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_refusals(cuda_device):
    q, k, v, g, state, _ = make(cuda_device, 10, 2, 4, 64, 64, BF, Hk=2)
    for bad in (lambda: la.linear_attention(q.cpu(), k, v, g), lambda: la.linear_attention(q.half(), k.half(), v.half(), g),
                lambda: la.linear_attention(q, k.float(), v, g), lambda: la.linear_attention(q, k[:9], v, g), lambda: la.linear_attention(q, k, v[:, :, :3], g[:, :, :3]),
                lambda: la.linear_attention(q, k, v, g[:9]), lambda: la.linear_attention(q, k, v, g.double()), lambda: la.linear_attention(q, k, v, g[0, 0, :3]),
                lambda: la.linear_attention(q, k, v, g, state.bfloat16()), lambda: la.linear_attention(q, k, v, g, state[:1]),
                lambda: la.linear_attention(q, k, v, g, lengths=torch.tensor([1, 2], device=cuda_device)), lambda: la.linear_attention(q, k, v, g, lengths=torch.ones(3, dtype=torch.int32, device=cuda_device)),
                lambda: la.linear_attention(q[0], k[0], v[0], g[0]), lambda: la.linear_attention_step(q, k, v, g, state),
                lambda: la.linear_attention_step(q[0], k[0], v[0], g[0], state.transpose(2, 3)), lambda: la.linear_attention_step(q[0], k[0], v[0], g[0], state[:1].expand(2, 4, 64, 64)),
                lambda: la.linear_attention_step(q[0], k[0], v[0], g[0], state[..., :32])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="head sizes"):
        la.linear_attention(*make(cuda_device, 3, 1, 1, 257, 8, F32)[:4])
    with pytest.raises(RuntimeError, match="no gradient"):
        la.linear_attention_step(q[0].clone().requires_grad_(), k[0], v[0], g[0], state)


@pytest.mark.parametrize("batch_first", [False, True])
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_layers_as_they_are_used(dtype, batch_first, cuda_device):
    """Two layers: a padded prompt, then tokens one by one; the same as the prompt and the tokens in one call."""
    torch.manual_seed(3)
    layers = [la.LinearAttention(96, 4, 32, 24, num_key_heads=2, batch_first=batch_first).to(cuda_device, dtype) for _ in range(2)]
    T, B = 150, 3
    x = torch.randn(T + 4, B, 96, device=cuda_device, dtype=dtype)
    cut = (lambda t: t.transpose(0, 1)) if batch_first else (lambda t: t)
    with torch.no_grad():
        def whole(t):
            y, stream, states = cut(t), None, []
            for layer in layers:
                y, stream, s = layer(y, stream)
                states.append(s)
            return cut(y), states
        want, want_states = whole(x)
        y, states = whole(x[:T])
        for t in range(T, T + 4):
            y, stream = x[t], None
            for layer, s in zip(layers, states):
                y, stream = layer.step(y, s, stream)
            # both are results of the type, a few roundings deep in the same places
            tol = 64 * ref.U[dtype] if dtype == BF else 4096 * ref.U[dtype]
            assert (y.float() - want[t].float()).abs().max() <= tol * want.float().abs().max()
    for s, w in zip(states, want_states):
        assert (s - w).norm() <= (64 * ref.U[dtype] if dtype == BF else 4096 * ref.U[dtype]) * w.norm()
    # a training step: every parameter gets a gradient
    lengths = torch.tensor([T, 0, 70], dtype=torch.int32, device=cuda_device)
    y, stream = cut(x[:T]).contiguous(), None
    for layer in layers:
        y, stream, s = layer(y, stream, lengths=lengths)
    (y.float().square().sum() + stream.float().square().sum() + s.square().sum()).backward()
    for layer in layers:
        for name, p in layer.named_parameters():
            assert p.grad is not None and torch.isfinite(p.grad).all() and p.grad.float().abs().max() > 0, name


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_broadcast_inputs_and_states_off_alignment(dtype, cuda_device):
    """One sequence of keys for all of the batch (a stride of 0), and a state that begins 4 bytes off."""
    q, k, v, g, state, _ = make(cuda_device, 140, 3, 2, 64, 64, dtype, decay=dtype)
    one = k[:, :1].clone().requires_grad_()
    off = torch.empty(state.numel() + 1, device=cuda_device)[1:].view(state.shape).copy_(state)
    leaves = [q.requires_grad_(), one, v.requires_grad_(), g.requires_grad_(), off.requires_grad_()]
    out, last = la.linear_attention(q, one.expand_as(q), v, g, off)
    dout, dstate = torch.randn_like(out), torch.randn_like(last)
    grads = torch.autograd.grad((out, last), leaves, (dout, dstate))
    want, bound = want_of(q.detach(), one.detach().expand_as(q), v.detach(), g.detach(), state, None, dout=dout, dstate=dstate)
    got = dict(zip(("dq", "dk", "dv", "dg", "dstate0"), grads))
    dk = got.pop("dk")
    hold({"out": out.detach(), "state": last.detach(), **got}, want, bound)
    # three results of the type, added in it: a rounding of the sum each
    size = want["dk"].abs().sum(1, keepdim=True)
    assert ((dk.double() - want["dk"].sum(1, keepdim=True)).abs() <= bound["dk"].sum(1, keepdim=True) + 3 * ref.U[dtype] * size).all()


def test_a_second_derivative_is_refused(cuda_device):
    q, k, v, g, state, _ = make(cuda_device, 20, 1, 1, 64, 64, F32)
    q.requires_grad_()
    dq, = torch.autograd.grad(la.linear_attention(q, k, v, g)[0].square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        dq.sum().backward()


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_a_captured_training_step(dtype, cuda_device):
    q, k, v, g, state, _ = make(cuda_device, 300, 2, 4, 64, 64, dtype, Hk=2, decay=dtype)
    leaves = [t.requires_grad_() for t in (q, k, v, g, state)]
    w = torch.randn(300, 2, 4, 64, device=cuda_device).to(dtype)

    def run():
        out, last = la.linear_attention(*leaves)
        return [out.detach(), *torch.autograd.grad((out, last), leaves, (w, torch.ones_like(last)))]

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = run()
    for _ in range(2):
        with torch.no_grad():
            q.mul_(-0.5)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(run(), got))


def test_threads(cuda_device):
    """Two threads, a stream and inputs each: nothing is shared."""
    import threading
    results, errors = {}, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                leaves = [t.requires_grad_() for t in make(cuda_device, 400, 2, 4, 64, 64, BF, decay=BF, seed=i)[:5]]
                for _ in range(20):
                    out, last = la.linear_attention(*leaves)
                    grads = torch.autograd.grad((out, last), leaves, (torch.ones_like(out), torch.ones_like(last)))
                torch.cuda.current_stream().synchronize()
                results[i] = [out.detach(), *grads]
        except Exception as e:       # (told below, in the test's own thread)
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    again = results.copy()
    for i in range(2):
        work(i)
        assert all(torch.equal(a, b) for a, b in zip(again[i], results[i]))


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_offsets_beyond_32_bits(dtype, cuda_device):
    """2.2e9 elements a tensor: the last sequences against the same in 64 bits."""
    T, B, H, D = (130, 8400, 16, 128) if dtype == BF else (130, 16500, 16, 64)

    def big():
        return torch.empty(T, B, H, D, dtype=dtype, device=cuda_device).normal_()

    q, k, v = big(), big(), big()
    g = torch.full((T, B, H), -0.1, device=cuda_device)
    out, last = la.linear_attention(q, k, v, g)
    part = [t[:, -2:].contiguous() for t in (q, k, v, g)]
    want, bound = want_of(*part, None, None)
    hold({"out": out[:, -2:], "state": last[-2:]}, want, bound)
    del q, k, v, g, out
    # a step of all of them, the last two with tokens of their own
    tokens = [torch.zeros(B, *t.shape[2:], dtype=t.dtype, device=cuda_device) for t in part]
    for t, x in zip(tokens, part):
        t[-2:] = x[0]
    want, bound = want_of(*[t[-2:][None] for t in tokens], last[-2:].clone(), None)
    out = la.linear_attention_step(*tokens, last)
    hold({"out": out[-2:][None], "state": last[-2:]}, want, bound)


def test_a_capture_beside_a_living_graph_is_refused(cuda_device):
    q, k, v, g, state, _ = make(cuda_device, 30, 2, 2, 64, 64, BF)
    leaves = [t.requires_grad_() for t in (q, k, v, g, state)]
    for only in range(5):
        use = [t if i == only else t.detach() for i, t in enumerate(leaves)]
        alive = la.linear_attention(*use)                       # on the default stream
        side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            something = torch.zeros(8, device=cuda_device)
            with pytest.raises(RuntimeError, match="still lives"):
                la.linear_attention(*use)
            with torch.no_grad():
                out, _ = la.linear_attention(*use)              # no gradient, nothing to refuse
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, alive[0]) and not something.any()
        del alive, graph


def test_a_state_that_must_not_be_written_is_left_alone(cuda_device):
    q, k, v, g, _, _ = make(cuda_device, 1, 2, 2, 64, 64, BF)
    with torch.inference_mode():
        state = torch.ones(2, 2, 64, 64, device=cuda_device)
    with pytest.raises(RuntimeError, match="[Ii]nference"):
        la.linear_attention_step(q[0], k[0], v[0], g[0], state)
    assert bool((state == 1).all())
    with torch.inference_mode():
        la.linear_attention_step(q[0], k[0], v[0], g[0], state)


@pytest.mark.parametrize("sizes", [(0, 2), (8, 0), (8, 4, 64, 64, 0), (8, 4, 0), (8, 4, 64, -1), (8, 4, 64, 64, 3)])
def test_layer_sizes(sizes):
    with pytest.raises(ValueError):
        la.LinearAttention(*sizes)


@pytest.mark.parametrize("case", [
    dict(H=8, Dk=64, Dv=64), dict(H=8, Dk=128, Dv=64, Hk=4), dict(H=8, Dk=64, Dv=128), dict(H=8, Dk=128, Dv=128, batch_first=True, fused=True),
    dict(H=8, Dk=60, Dv=60), dict(H=8, Dk=100, Dv=128, Hk=2),
], ids=lambda c: "-".join(f"{k}{v}" for k, v in c.items()))
def test_more_chunks_than_multiprocessors(case, cuda_device):
    T, B = 200, 45                     # 720 chunks, of which some are whole, some short, some behind the end of their sequence
    lengths = [(0, 1, 127, 128, 129, 200, 63, 128, 200)[b % 9] for b in range(B)]
    q, k, v, g, state, n = make(cuda_device, T, B, dtype=BF, decay=BF, lengths=lengths, **case)
    bf = case.get("batch_first", False)
    leaves = [t.detach().requires_grad_() for t in (q, k, v, g, state)]
    out, last = la.linear_attention(*leaves, lengths=n, batch_first=bf)
    dout, dstate = torch.randn_like(out), torch.randn_like(last)
    grads = torch.autograd.grad((out, last), leaves, (dout, dstate), retain_graph=True)
    want, bound = want_of(q, k, v, g, state, n, bf, dout=dout, dstate=dstate)
    hold({"out": out, "state": last, **dict(zip(("dq", "dk", "dv", "dg", "dstate0"), grads))}, want, bound)
    for _ in range(20):
        again = torch.autograd.grad((out, last), leaves, (dout, dstate), retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(grads, again))
