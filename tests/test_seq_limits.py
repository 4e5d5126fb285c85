"""The limits that the sequence operators' results are held to are tight enough to miss what they are there for."""
import pytest
import torch

from tests import seq_reference as ref
from tests import seq_terms as terms


def positive(T, B, H, Dk, Dv, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    q, k, v, dout = ((torch.randn(T, B, H, d, generator=gen).abs() + 0.1).to(dtype) for d in (Dk, Dk, Dv, Dv))
    g = -torch.nn.functional.softplus(torch.randn(T, B, H, generator=gen) - torch.linspace(1.0, 7.0, H))
    state, dstate = (torch.randn(B, H, Dk, Dv, generator=gen).abs() for _ in range(2))
    return q, k, v, g, state, dout, dstate


@pytest.mark.parametrize("dtype,chunk", [(torch.bfloat16, 128), (torch.float32, 64)], ids=["bf16", "fp32"])
@pytest.mark.parametrize("Dk,Dv", [(64, 64), (64, 128), (128, 64), (128, 128)])
def test_a_missing_term_of_the_decays_gradient_is_noticed(Dk, Dv, dtype, chunk):
    q, k, v, g, state, dout, dstate = positive(300, 1, 2, Dk, Dv, dtype)
    want = ref.attention(q, k, v, g, state, None, None, dout, dstate)
    d, types = terms.attention_limits(want, q, k, v, g, state, None, dout, dstate)
    whole = terms.decays_gradient(q, k, v, g, state, dout, dstate, chunk)
    assert ((whole - want["dg"]).abs() <= 1e-10 * want["dg"]).all()
    assert terms.off_of(whole, want["dg"], d["dg"], types["dg"]) <= 1
    for name in terms.DECAY_TERMS:
        part = terms.decays_gradient(q, k, v, g, state, dout, dstate, chunk, without=name)
        assert terms.off_of(part, want["dg"], d["dg"], types["dg"]) > 10, name


@pytest.mark.parametrize("T,D", terms.SHORT, ids=str)
def test_a_missing_third_part_of_a_state_is_noticed(T, D):
    gen = torch.Generator().manual_seed(T)
    k, v = torch.randn(T, 4, 4, D[0], generator=gen).bfloat16(), torch.randn(T, 4, 4, D[1], generator=gen).bfloat16()
    G = (-0.1 * torch.rand(T, 4, 4, generator=gen)).cumsum(0)
    w = (G[-1] - G).exp()
    x, parts = k.float() * w[..., None], []
    for _ in range(3):
        parts.append(x.bfloat16())
        x = x - parts[-1].float()
    want, size = (torch.einsum("tbhi,tbhj->bhij", a, b) for a, b in ((k.double() * w.double()[..., None], v.double()), (k.double().abs() * w.double()[..., None], v.double().abs())))
    off = []
    for n in (2, 3):
        got = torch.einsum("tbhi,tbhj->bhij", sum(p.double() for p in parts[:n]), v.double())
        off.append(((got - want).abs() / terms.short_state_limit(size, T)).max())
    assert off[0] > 2 and off[1] < 0.5
