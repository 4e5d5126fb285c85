"""Linear attention in bf16: nothing inside is coarser than 16 bits, so a result is its type's rounding of a sum that is nearly exact.

A factor of a product on the tensor cores is one bf16 value or the sum of two or three.  Two parts: the first is off by 2^-8 of the factor
at the most (half a step), the second by 2^-8 of what is left: 2^-16 of the factor.  So held are the pairs' weights (P, E), the
state before a chunk and its gradient behind it, one of them in a product; k times its decays, three parts, is as good as
fp32.  Sums are fp32, n terms one after the other: n 2^-24 of the sum of the terms' sizes.  With d = (2^-16 + n 2^-24) size a sum is off by d at the most;
its rounding to the type is a nearest one, whose distance from the grid changes by no more than the sum does, so the result is off by
|round(want) - want| + 2 d."""
import pytest
import torch

from tests import seq_reference as ref
from tests.test_gpu_linear_attention import BF, F32, la, make

pytestmark = pytest.mark.gpu
F = 2.0 ** -24


def limits(want, q, k, v, g, state, n, dout, dstate):
    """name -> how far it may be off, for time-first arguments with heads repeated."""
    sizes = ref.attention(q.abs(), k.abs(), v.abs(), g, state.abs() if state is not None else None, n, None, dout.abs(), dstate.abs())
    terms = q.shape[0] + 2 * max(q.shape[-1], v.shape[-1]) + 24
    types = {"state": F32, "dstate0": F32, "dg": g.dtype}
    d = {name: ((0 if types.get(name) == F32 and name != "dg" else 2.0 ** -16) + terms * F) * size for name, size in sizes.items()}
    # the decays' gradient is a running sum of what cancels in a chunk
    qdq, kdk = (q.double().abs() * sizes["dq"]).sum(-1), (k.double().abs() * sizes["dk"]).sum(-1)
    d["dg"] = 2.0 ** -16 * sizes["dg"] + terms * F * (sizes["dg"] + (qdq + kdk).flip(0).cumsum(0).flip(0))
    return d, {name: types.get(name, BF) for name in sizes}


def shared(x, heads):
    return x.unflatten(2, (heads, -1)).sum(3)


CASES = [dict(T=300, B=2, H=2, Dk=64, Dv=64), dict(T=300, B=2, H=2, Dk=128, Dv=64), dict(T=300, B=2, H=2, Dk=64, Dv=128), dict(T=300, B=2, H=2, Dk=128, Dv=128),
         dict(T=1000, B=1, H=2, Dk=128, Dv=128, fused=True), dict(T=260, B=3, H=4, Dk=64, Dv=64, Hk=2, lengths=[260, 129, 77]), dict(T=200, B=2, H=2, Dk=128, Dv=130),
         dict(T=24, B=1, H=4, Dk=64, Dv=64), dict(T=128, B=2, H=2, Dk=60, Dv=60, h0=False),
         dict(T=300, B=2, H=2, Dk=60, Dv=60), dict(T=200, B=2, H=2, Dk=100, Dv=128, Hk=1), dict(T=200, B=2, H=2, Dk=33, Dv=17, lengths=[200, 130])]


def check(got, want, d, types, Hk):
    for name, x in got.items():
        w, s = (shared(want[name], Hk), shared(d[name], Hk)) if name in ("dq", "dk") else (want[name], d[name])
        off = (x.double() - w).abs() / ((w.to(types[name]).double() - w).abs() + 2 * s + 1e-30)
        assert off.max() <= 1, f"{name}: {off.max():.2f} times the limit, at {[int(i) for i in (off == off.max()).nonzero()[0]]}"


@pytest.mark.parametrize("decay", [F32, BF], ids=["fp32_decays", "bf16_decays"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(f"{k}{v}" for k, v in c.items()))
def test_outputs_are_nearly_their_types_roundings(case, decay, cuda_device):
    q, k, v, g, state, n = make(cuda_device, dtype=BF, decay=decay, **case)
    H, Hk = v.shape[2], q.shape[2]
    out, last = la.linear_attention(q, k, v, g, state, n)
    args = [x.repeat_interleave(H // Hk, 2) for x in (q, k)] + [v, g]
    zeros = torch.zeros_like(out), torch.zeros_like(last)
    want = ref.attention(*args, state=state, lengths=n)
    d, types = limits(want, *args, state, n, *zeros)
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
    d, types = limits(want, *args, state, n, dout, dstate)
    check(got, want, d, types, Hk)
    with torch.no_grad():        # the form that keeps no states for a gradient
        again = la.linear_attention(q, k, v, g, state, n)
    assert torch.equal(again[0], out) and torch.equal(again[1], last)
