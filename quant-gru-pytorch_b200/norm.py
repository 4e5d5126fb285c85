"""Root-mean-square norm with the residual's addition, in one pass over the row: what stands between the layers of a stack
(no counterpart in the reference).

``rms_norm``     y = h * weight / sqrt(mean(h^2) + eps) with h = x + residual; differentiable
``rms_norm_q8``  the same with y in 8 bits: with a scale for each row, or with the scale and zero point of an
                 operator that has been calibrated, as ``QuantGRU.forward_quantized`` takes its input

Tensors are float32 or bfloat16 on the GPU, rows of up to 16384 features; arguments are checked, memory is allocated and the library
is called in csrc/qgru_seq_torch.cc.  Everything runs on the current stream of the tensors' device and waits for nothing.
Inputs with a forward-mode tangent are refused, by ``rms_norm_q8`` where the residual's stream has one.
"""
from . import _cabi


def rms_norm(x, weight, residual=None, eps=1e-6):
    """x [..., D], weight [D], residual like x or None.  Returns y, or with a residual (y, h): h = x + residual, rounded to
    their type, is the stream that goes on to the next addition, and y is the norm of what is stored."""
    return (_cabi._seq or _cabi.seq()).rms_norm(x, weight, residual, eps)


def rms_norm_q8(x, weight, residual=None, eps=1e-6, scale=None, zero_point=0, bits=8, unsigned=False):
    """The norm's output in 8 bits, without a gradient (refused where the residual's stream has one).

    With ``scale=None`` every row has a scale of its own: returns (q int8, scales [...] float32[, h]) with q * scale the
    norm, |q| <= 127 (a row of zeros: 0 and 0; a row with infinities or NaN: 0 and NaN).  With a scale (and zero point, width
    and sign, as the input operator of a calibrated layer has them) returns q, or (q, h): q = clamp(round(y / scale) + zero_point)
    in int8, or uint8 where ``unsigned``.  Halves round to even."""
    return (_cabi._seq or _cabi.seq()).rms_norm_q8(x, weight, residual, eps, scale, zero_point, bits, unsigned)
