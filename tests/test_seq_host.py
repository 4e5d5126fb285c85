"""What the sequence operators refuse before anything reaches a GPU."""
import ctypes as C
import importlib

import pytest
import torch

from __graft_entry__ import PKG_NAME

_cabi = importlib.import_module(PKG_NAME + "._cabi")
la = importlib.import_module(PKG_NAME + ".linear_attention")
norm = importlib.import_module(PKG_NAME + ".norm")


def attention(**kw):
    a = _cabi.Attention()
    for name, value in {**dict(T=4, B=2, H=4, Hk=2, Dk=64, Dv=64, scale=1.0), **kw}.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("bad", [dict(T=-1), dict(B=-1), dict(H=0), dict(Hk=0), dict(Dk=0), dict(Dv=0), dict(Hk=3)], ids=str)
def test_attention_sizes_are_checked(bad):
    L = _cabi.lib()
    a = attention(**bad)
    assert L.qgru_attention_sizes(a, None, None, None) == _cabi.QGRU_ERR_BAD_ARG
    assert L.qgru_attention_forward(a, None) == L.qgru_attention_backward(a, None) == _cabi.QGRU_ERR_BAD_ARG
    assert L.qgru_attention_step(a, 0, 0, None) == _cabi.QGRU_ERR_BAD_ARG
    assert L.qgru_seq_last_error()


def test_what_the_kernels_do_not_take():
    L = _cabi.lib()
    for bad in (dict(Dk=257), dict(Dv=300), dict(T=(1 << 30) + 1), dict(B=1 << 20, H=1 << 12, Hk=1 << 12)):
        assert L.qgru_attention_forward(attention(**bad), None) == _cabi.QGRU_ERR_UNSUPPORTED
    assert L.qgru_attention_forward(None, None) == L.qgru_norm_forward(None, None) == _cabi.QGRU_ERR_BAD_ARG
    n = _cabi.Norm(cols=16385, rows=1)
    assert L.qgru_norm_forward(n, None) == _cabi.QGRU_ERR_UNSUPPORTED
    assert b"16385" in L.qgru_seq_last_error()
    for bad in (_cabi.Norm(cols=0, rows=1), _cabi.Norm(cols=4, rows=-1), _cabi.Norm(cols=4, rows=1)):
        assert L.qgru_norm_forward(bad, None) == _cabi.QGRU_ERR_BAD_ARG
    assert L.qgru_norm_forward(_cabi.Norm(cols=4, rows=0), None) == 0
    assert L.qgru_attention_step(attention(), 0, 0, None) == _cabi.QGRU_ERR_BAD_ARG          # null tensors
    assert L.qgru_attention_forward(attention(B=0), None) == 0


def test_given_scale_is_a_range_of_eight_bits():
    L = _cabi.lib()
    for lo, hi in ((-129, 0), (0, 256), (-1, 128), (3, 2)):
        n = _cabi.Norm(cols=4, rows=1, x=16, weight=16, q8=16, q8_scale=0.5, q8_lo=lo, q8_hi=hi)
        assert L.qgru_norm_forward(n, None) == _cabi.QGRU_ERR_BAD_ARG
        assert str(lo).encode() in L.qgru_seq_last_error()


def test_struct_layout():
    assert C.sizeof(_cabi.SeqTensor) == 32
    assert C.sizeof(_cabi.Attention) == 12 * 4 + 7 * 8 + 2 * 8 + 10 * 32
    assert C.sizeof(_cabi.Norm) == 16 + 8 + 8 + 3 * 8 + 16 + 16 + 16 + 24 + 16


def test_host_tensors_are_refused():
    x = torch.zeros(3, 2, 4, 8)
    with pytest.raises(ValueError, match="CUDA"):
        la.linear_attention(x, x, x, torch.zeros(3, 2, 4))
    with pytest.raises(ValueError, match="CUDA"):
        la.linear_attention_step(x[0], x[0], x[0], torch.zeros(2, 4), torch.zeros(2, 4, 8, 8))
    with pytest.raises(ValueError, match="CUDA"):
        norm.rms_norm(x, torch.ones(8))
    with pytest.raises(ValueError, match="share"):
        la.LinearAttention(32, 4, num_key_heads=3)
