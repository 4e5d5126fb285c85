"""Linear attention: nothing inside is coarser than 16 bits (fp32 for fp32), so a result is its type's rounding of a sum that is nearly exact
(tests/seq_terms.py says how near)."""
import pytest
import torch

from tests import seq_reference as ref
from tests import seq_terms as terms
from tests.seq_terms import attention_limits
from tests.test_gpu_linear_attention import BF, F32, la, make
from tests.test_seq_limits import positive

pytestmark = pytest.mark.gpu


def shared(x, heads):
    return x.unflatten(2, (heads, -1)).sum(3)


CASES = [dict(T=300, B=2, H=2, Dk=64, Dv=64), dict(T=300, B=2, H=2, Dk=128, Dv=64), dict(T=300, B=2, H=2, Dk=64, Dv=128), dict(T=300, B=2, H=2, Dk=128, Dv=128),
         dict(T=1000, B=1, H=2, Dk=128, Dv=128, fused=True), dict(T=260, B=3, H=4, Dk=64, Dv=64, Hk=2, lengths=[260, 129, 77]), dict(T=200, B=2, H=2, Dk=128, Dv=130),
         dict(T=24, B=1, H=4, Dk=64, Dv=64), dict(T=128, B=2, H=2, Dk=60, Dv=60, h0=False),
         dict(T=300, B=2, H=2, Dk=60, Dv=60), dict(T=200, B=2, H=2, Dk=100, Dv=128, Hk=1), dict(T=200, B=2, H=2, Dk=33, Dv=17, lengths=[200, 130])]


def check(got, want, d, types, Hk):
    for name, x in got.items():
        w, s = (shared(want[name], Hk), shared(d[name], Hk)) if name in ("dq", "dk") else (want[name], d[name])
        off = terms.off_of(x, w, s, types[name])
        assert off <= 1, f"{name}: {off:.2f} times the limit"


@pytest.mark.parametrize("decay", [F32, BF], ids=["fp32_decays", "bf16_decays"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(f"{k}{v}" for k, v in c.items()))
def test_outputs_are_nearly_their_types_roundings(case, decay, cuda_device):
    q, k, v, g, state, n = make(cuda_device, dtype=BF, decay=decay, **case)
    H, Hk = v.shape[2], q.shape[2]
    out, last = la.linear_attention(q, k, v, g, state, n)
    args = [x.repeat_interleave(H // Hk, 2) for x in (q, k)] + [v, g]
    want = ref.attention(*args, state=state, lengths=n)
    d, types = attention_limits(want, *args, state, n)
    check({"out": out, "state": last}, want, d, types, Hk)


@pytest.mark.parametrize("decay", [F32, BF], ids=["fp32_decays", "bf16_decays"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(f"{k}{v}" for k, v in c.items()))
def test_gradients_are_nearly_their_types_roundings(case, decay, cuda_device):
    q, k, v, g, state, n = make(cuda_device, dtype=BF, decay=decay, **case)
    H, Hk = v.shape[2], q.shape[2]
    names = ["dq", "dk", "dv", "dg"] + (["dstate0"] if state is not None else [])
    leaves = [t.detach().requires_grad_() for t in (q, k, v, g, state) if t is not None]
    out, last = la.linear_attention(*leaves, lengths=n)
    dout, dstate = torch.randn_like(out), torch.randn_like(last)
    got = dict(zip(names, torch.autograd.grad((out, last), leaves, (dout, dstate))))
    args = [x.repeat_interleave(H // Hk, 2) for x in (q, k)] + [v, g]
    want = ref.attention(*args, state=state, lengths=n, dout=dout, dstate=dstate)
    d, types = attention_limits(want, *args, state, n, dout, dstate)
    check(got, want, d, types, Hk)
    with torch.no_grad():        # the form that keeps no states for a gradient
        again = la.linear_attention(q, k, v, g, state, n)
    assert torch.equal(again[0], out) and torch.equal(again[1], last)


@pytest.mark.parametrize("decay", [F32, BF], ids=["fp32_decays", "bf16_decays"])
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("Dk,Dv", [(64, 64), (64, 128), (128, 64), (128, 128), (60, 60), (33, 100), (200, 256)])
def test_gradients_of_terms_that_do_not_cancel(Dk, Dv, dtype, decay, cuda_device):
    """All positive: a limit is a part of the value itself, and no term of the decays' gradient can be missing."""
    if dtype == F32 and decay == BF:
        pytest.skip("decays are float32 or the type of q")
    q, k, v, g, state, dout, dstate = (t.to(cuda_device) for t in positive(300, 1, 2, Dk, Dv, dtype))
    g = g.to(decay)
    leaves = [t.requires_grad_() for t in (q, k, v, g, state)]
    out, last = la.linear_attention(*leaves)
    got = dict(zip(("dq", "dk", "dv", "dg", "dstate0"), torch.autograd.grad((out, last), leaves, (dout, dstate))))
    args = [t.detach() for t in leaves[:4]]
    want = ref.attention(*args, state=state.detach(), dout=dout, dstate=dstate)
    d, types = attention_limits(want, *args, state.detach(), None, dout, dstate)
    check({"out": out.detach(), "state": last.detach(), **got}, want, d, types, 2)


@pytest.mark.parametrize("T,D", terms.SHORT, ids=str)
def test_states_of_a_few_tokens_have_24_bits(T, D, cuda_device):
    """k times its decays, or q from the end, is three bf16 parts on the tensor cores, whichever kernel takes the size."""
    q, k, v, _, _, _ = make(cuda_device, T, 4, 4, *D, BF, seed=T)
    dout, g = torch.randn_like(v), -0.1 * torch.rand(T, 4, 4, device=cuda_device)
    state = torch.zeros(4, 4, *D, device=cuda_device, requires_grad=True)
    out, last = la.linear_attention(q, k, v, g, state)
    dstate0, = torch.autograd.grad(out, state, dout)
    want = ref.attention(q, k, v, g, dout=dout)
    sizes = ref.attention(q.abs(), k.abs(), v.abs(), g, dout=dout.abs())
    for name, x in (("state", last), ("dstate0", dstate0)):
        off = ((x.double() - want[name]).abs() / terms.short_state_limit(sizes[name], T)).max()
        assert off <= 1, f"{name}: {off:.2f} times the limit"
