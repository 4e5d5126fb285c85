"""Sequence operators where a value that does not count, an order of arrival or a caller's mode could reach a result."""
import importlib

import pytest
import torch

from __graft_entry__ import PKG_NAME
from tests import seq_reference as ref
from tests.test_gpu_linear_attention import hold, make, want_of

la = importlib.import_module(PKG_NAME + ".linear_attention")
norm = importlib.import_module(PKG_NAME + ".norm")
pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("Dk,Dv", [(128, 64), (96, 40), (128, 128), (64, 64)])
def test_short_chunks_behind_whole_ones(Dk, Dv, cuda_device):
    """Many chunks a CTA whose keys come out of L2 (shared by all heads) and whose values do not: whatever arrives first, the rows behind
    a sequence are cleared in the chunk that they belong to."""
    T, B, H = 500, 90, 8
    lengths = [(1, 129, 500, 0, 257, 385, 500, 130)[b % 8] for b in range(B)]
    q, k, v, g, state, n = make(cuda_device, T, B, H, Dk, Dv, BF, Hk=1, lengths=lengths, decay=BF)
    past = torch.arange(T, device=cuda_device)[:, None] >= n[None, :]
    want = la.linear_attention(*[torch.where(past[(...,) + (None,) * (t.dim() - 2)], 0.0, t) for t in (q, k, v, g)], state, n)
    for t in (q, k, g):
        t[past] = float("nan")
    v[past] = float("inf")
    for _ in range(20):
        got = la.linear_attention(q, k, v, g, state, n)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    part = slice(0, 8)
    clean = [torch.where(past[:, part][(...,) + (None,) * (t.dim() - 2)], 0.0, t[:, part]) for t in (q, k, v, g)]
    exact, bound = want_of(*clean, state[part], n[part])
    hold({"out": want[0][:, part], "state": want[1][part]}, exact, bound)


@pytest.mark.parametrize("dtype,Dk,Dv", [(F32, 128, 128), (BF, 200, 256), (F32, 72, 40), (F32, 64, 64), (BF, 128, 128), (BF, 60, 60)], ids=str)
def test_one_infinite_value_at_each_token_of_a_chunk(dtype, Dk, Dv, cuda_device):
    """Sequence b has a single infinity, at token b of its last chunk: no earlier output knows of it."""
    C = 128 if dtype == BF and Dk <= 128 else 64
    T = 2 * C
    q, k, v, g, state, _ = make(cuda_device, T, C, 1, Dk, Dv, dtype, seed=5)
    want, bound = want_of(q, k, v, g, state, None)
    at = torch.arange(C, device=cuda_device)
    v[C + at, at, 0, (7 * at) % Dv] = float("inf")
    before = torch.arange(T, device=cuda_device)[:, None] < C + at[None, :]
    for _ in range(20):
        out = la.linear_attention(q, k, v, g, state)[0]
        assert torch.isfinite(out[before]).all()
        hold({"out": out[before]}, {"out": want["out"][before]}, {"out": bound["out"][before]})
        assert not torch.isfinite(out[C + at, at, 0, (7 * at) % Dv]).any()


def test_inputs_with_a_tangent_are_refused(cuda_device):
    import torch.autograd.forward_ad as fwd
    q, k, v, g, state, _ = make(cuda_device, 20, 2, 2, 64, 64, F32)
    x, w, r = torch.randn(3, 64, device=cuda_device), torch.ones(64, device=cuda_device), torch.randn(3, 64, device=cuda_device)
    token = [t[0].clone() for t in (q, k, v, g)] + [state.clone()]
    calls = [(la.linear_attention, [q, k, v, g, state]), (la.linear_attention, [q, k, v, g[0, 0].clone(), state]), (la.linear_attention_step, token), (norm.rms_norm, [x, w]),
             (norm.rms_norm, [x, w, r])]
    for call, args in calls:
        for i in range(len(args)):
            for grad in (False, True):
                with fwd.dual_level(), torch.set_grad_enabled(grad):
                    use = [fwd.make_dual(t, torch.ones_like(t)) if i == j else t for j, t in enumerate(args)]
                    with pytest.raises(NotImplementedError, match="forward-mode"):
                        call(*use)
                    call(*[fwd.unpack_dual(t).primal for t in use])
    before = token[4].clone()
    for i in (0, 2):
        with fwd.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
            use = [fwd.make_dual(t, t) if i == j else t for j, t in enumerate([x, w, r])]
            norm.rms_norm_q8(*use)
    with fwd.dual_level():
        norm.rms_norm_q8(x, fwd.make_dual(w, w), r)            # a layer's weight alone has no part in the stream
        with pytest.raises(NotImplementedError, match="forward-mode"):
            la.linear_attention_step(*token[:4], fwd.make_dual(token[4], token[4]))
    assert torch.equal(token[4], before)
    layer = la.LinearAttention(64, 2, 32, 32).to(cuda_device)
    with pytest.raises(Exception):
        torch.func.jvp(lambda t: layer(t)[0], (torch.randn(5, 2, 64, device=cuda_device),), (torch.ones(5, 2, 64, device=cuda_device),))


_cabi = importlib.import_module(PKG_NAME + "._cabi")


@pytest.fixture
def expire(cuda_device):
    """As a kernel leaves it whose wait has run out; nothing of it stays."""
    def nothing_told():                  # (to this thread, nor to the one that runs backward passes)
        leaf = torch.ones(1, 8, device=cuda_device, requires_grad=True)
        for _ in range(3):
            try:
                norm.rms_norm(leaf, leaf[0]).sum().backward()
            except RuntimeError as e:
                assert "run out" in str(e)

    nothing_told()
    yield lambda: _cabi.check(_cabi.lib().qgru_seq_test_expire(0), "qgru_seq_test_expire")
    nothing_told()


def raises_expiry():
    return pytest.raises(_cabi.QgruError, match="run out")


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_whichever_call_comes_next_tells_that_a_wait_ran_out(dtype, expire, cuda_device):
    q, k, v, g, state, _ = make(cuda_device, 20, 2, 2, 64, 64, dtype)
    x, w, r = torch.randn(3, 64, device=cuda_device), torch.ones(64, device=cuda_device), torch.randn(3, 64, device=cuda_device)
    wide = make(cuda_device, 20, 2, 2, 200, 64, dtype)[:5]
    before = state.clone()
    for call in (lambda: la.linear_attention(q, k, v, g, state), lambda: la.linear_attention(*wide), lambda: la.linear_attention_step(q[0], k[0], v[0], g[0], state),
                 lambda: norm.rms_norm(x, w), lambda: norm.rms_norm(x, w, r), lambda: norm.rms_norm_q8(x, w), lambda: la.synchronize(), lambda: la.synchronize("cuda:0")):
        expire()
        with raises_expiry() as e:
            call()
        assert e.value.status == _cabi.QGRU_ERR_TIMEOUT
        assert torch.equal(state, before)            # nothing was queued
        call()                                       # told once
        state.copy_(before)
    leaf = q.detach().requires_grad_()
    out, _ = la.linear_attention(leaf, k, v, g)
    expire()
    with pytest.raises(RuntimeError, match="run out"):          # (what a node throws is a RuntimeError when the engine hands it on)
        torch.autograd.grad(out.sum(), leaf)


def test_every_thread_is_told_of_a_wait_that_ran_out(expire, cuda_device):
    """The one that finds it, and each that had work on the device; a thread whose first call comes later is not."""
    import threading
    q, k, v, g, state, _ = make(cuda_device, 20, 2, 2, 64, 64, BF)
    begun, go, told = threading.Barrier(3), threading.Event(), []

    def work(i):
        la.linear_attention(q, k, v, g, state)
        begun.wait()
        go.wait()
        for _ in range(3):
            try:
                la.linear_attention(q, k, v, g, state)
            except _cabi.QgruError:
                told.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    begun.wait()
    expire()
    with raises_expiry():
        la.linear_attention(q, k, v, g, state)
    go.set()
    for t in threads:
        t.join()
    assert sorted(told) == [0, 1]
    fresh = []

    def late():
        try:
            la.linear_attention(q, k, v, g, state)
            fresh.append("ran")
        except _cabi.QgruError:
            fresh.append("told")

    t = threading.Thread(target=late)
    t.start()
    t.join()
    assert fresh == ["ran"]


def hooked(change):
    """One saved tensor after the other comes back changed; how many there are is in `count`."""
    count = []

    def pack(t):
        count.append(t)
        return len(count) - 1

    return count, lambda only: torch.autograd.graph.saved_tensors_hooks(pack, lambda i: change(count[i]) if i == only else count[i])


@pytest.mark.parametrize("change", [lambda t: t[..., :-1], lambda t: t.to(torch.float64), lambda t: t.cpu(), lambda t: t.flatten()[: t.numel() // 2], lambda t: t[None]],
                         ids=["shorter", "double", "host", "half", "dimension"])
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_a_saved_tensor_that_comes_back_as_another_is_refused(dtype, change, cuda_device):
    q, k, v, g, state, n = make(cuda_device, 150, 2, 2, 64, 64, dtype, lengths=[150, 40], decay=dtype)
    x, r, w = torch.randn(6, 64, device=cuda_device).to(dtype), torch.randn(6, 64, device=cuda_device).to(dtype), torch.ones(64, device=cuda_device).to(dtype)
    for call, args, saves in ((lambda *a: la.linear_attention(*a, lengths=n)[0], (q, k, v, g, state), 6), (lambda *a: norm.rms_norm(*a)[0], (x, w, r), 3), (norm.rms_norm, (x, w), 3)):
        for only in range(saves):
            leaves = [t.detach().requires_grad_() for t in args]
            count, hooks = hooked(change)
            with hooks(only):
                out = call(*leaves)
            assert len(count) == saves
            with pytest.raises(RuntimeError, match="saved-tensor hook"):
                torch.autograd.grad(out.float().sum(), leaves)
    # lengths that come back in every second place of a larger tensor are still the lengths
    leaves = [t.detach().requires_grad_() for t in (q, k, v, g, state)]
    want = torch.autograd.grad(la.linear_attention(*leaves, lengths=n)[0].float().sum(), leaves)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: torch.stack([t, t + 7], -1)[..., 0] if t.dtype == torch.int32 else t):
        out = la.linear_attention(*leaves, lengths=n)[0]
    assert all(torch.equal(a, b) for a, b in zip(want, torch.autograd.grad(out.float().sum(), leaves)))


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("D", [8, 64, 128, 200])
def test_the_largest_values_are_values(D, dtype, cuda_device):
    """One factor of the largest finite value (or close to it), the others small: results are finite and as near as any."""
    most = torch.finfo(dtype).max
    for which in range(3):
        q, k, v, g, state, _ = make(cuda_device, 70, 2, 1, D, D, dtype, memory=(4.0, 4.0), h0=False)
        for i, t in enumerate((q, k, v)):
            t.mul_(2.0 ** -12)
            if i == which:
                t[3::17, 0, 0, 0] = most
                t[5::17, 1, 0, D - 1] = -most * (1 - 2.0 ** -12)
        args = (q, k, v, g)
        leaves = [t.detach().requires_grad_() for t in args]
        out, last = la.linear_attention(*leaves)
        want, bound = want_of(*args, None, None, dout=torch.full_like(out, 2.0 ** -30), dstate=torch.zeros_like(last))
        grads = torch.autograd.grad(out, leaves[:3], torch.full_like(out, 2.0 ** -30))
        hold({"out": out.detach(), "state": last.detach(), **dict(zip(("dq", "dk", "dv"), grads))}, want, bound)


@pytest.mark.parametrize("which", range(3), ids="qkv")
def test_infinities_of_a_single_token(which, cuda_device):
    """fp32: the product's infinity, with its sign, and not NaN."""
    for sign in (1.0, -1.0):
        for shape in ((1, 1), (1, 40), (1, 100)):
            q, k, v, g, _, _ = make(cuda_device, 1, 3, 2, *shape, F32, h0=False)
            (q, k, v)[which][:] = sign * float("inf")
            out, last = la.linear_attention(q, k, v, g)
            want, _ = want_of(q, k, v, g, None, None)
            assert torch.equal(out, want["out"].float()) and not out.isfinite().any() and not out.isnan().any()
            if which:
                assert torch.equal(last, want["state"].float())


@pytest.mark.parametrize("case", [dict(Dk=64, Dv=64), dict(Dk=128, Dv=64), dict(Dk=64, Dv=128, Hk=4), dict(Dk=128, Dv=128), dict(Dk=128, Dv=128, Hk=2), dict(Dk=100, Dv=127)],
                         ids=lambda c: "-".join(f"{k}{v}" for k, v in c.items()))
def test_the_same_bits_beside_other_work(case, cuda_device):
    """Many chunks a CTA while another stream keeps the memory and the multiprocessors busy: products and copies end in other orders, results do not."""
    T, B = 700, 37
    lengths = [min(T, (0, 1, 127, 128, 129, 200, 63, T, T, 385, 513)[b % 11]) for b in range(B)]
    q, k, v, g, state, n = make(cuda_device, T, B, 8, dtype=BF, lengths=lengths, decay=BF, **case)
    dout, dstate = torch.randn_like(v), torch.randn_like(state)

    def run():
        leaves = [t.detach().requires_grad_() for t in (q, k, v, g, state)]
        out, last = la.linear_attention(*leaves, lengths=n)
        return [out.detach(), last.detach(), *torch.autograd.grad((out, last), leaves, (dout, dstate))]

    other, a, b = torch.cuda.Stream(), torch.randn(2048, 2048, device=cuda_device), torch.empty(300_000_000, dtype=torch.uint8, device=cuda_device)
    want = run()
    for i in range(60):
        with torch.cuda.stream(other):
            if i % 3 == 0:
                a @ a
            elif i % 3 == 1:
                b.fill_(i)
        assert all(torch.equal(x, y) for x, y in zip(run(), want)), i
    torch.cuda.synchronize()
