"""Root-mean-square norm with the residual's addition, in one pass over the row: what stands between the layers of a stack
(no counterpart in the reference).

``rms_norm``     y = h * weight / sqrt(mean(h^2) + eps) with h = x + residual; differentiable
``rms_norm_q8``  the same with y in 8 bits: with a scale for each row, or with the scale and zero point of an
                 operator that has been calibrated, as ``QuantGRU.forward_quantized`` takes its input

Everything runs on the current stream of the tensors' device and waits for nothing.
"""
import torch
from torch.autograd.function import once_differentiable

from . import _cabi

_TYPES = (torch.float32, torch.bfloat16)


def _checked(x, weight, residual):
    if not isinstance(x, torch.Tensor) or not x.is_cuda or x.dtype not in _TYPES:
        raise ValueError("x must be a CUDA tensor of float32 or bfloat16")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must have at least one feature, got shape {list(x.shape)}")
    if not isinstance(weight, torch.Tensor) or weight.device != x.device or weight.dtype not in _TYPES:
        raise ValueError(f"weight must be a tensor of float32 or bfloat16 on {x.device}")
    if tuple(weight.shape) != (x.shape[-1],):
        raise ValueError(f"weight must have shape {[x.shape[-1]]}, got {list(weight.shape)}")
    if residual is not None and (not isinstance(residual, torch.Tensor) or residual.device != x.device or residual.dtype != x.dtype or residual.shape != x.shape):
        raise ValueError(f"residual must be a {x.dtype} tensor of shape {list(x.shape)} on {x.device}")


def _rows(t):
    """A tensor as rows: [n, features], features next to each other (a copy where its strides do not allow a view)."""
    t = t.reshape(-1, t.shape[-1]) if t.numel() else t.new_empty((0, t.shape[-1]))
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 and t.is_contiguous() else t.contiguous()


def _call(x2, weight, r2, eps, h, y=None, q8=None, scales=None, rstd=None, given=None):
    scale, zero_point, lo, hi = given or (0.0, 0, 0, 0)
    n = _cabi.Norm(x2.device.index or 0, x2.dtype == torch.bfloat16, weight.dtype == torch.bfloat16, x2.shape[1], x2.shape[0], eps,
                   x2.data_ptr(), r2.data_ptr() if r2 is not None else None, weight.data_ptr(), x2.stride(0), r2.stride(0) if r2 is not None else 0,
                   h.data_ptr() if h is not None else None, y.data_ptr() if y is not None else None, x2.shape[1], x2.shape[1],
                   q8.data_ptr() if q8 is not None else None, scales.data_ptr() if scales is not None else None,
                   rstd.data_ptr() if rstd is not None else None, scale, zero_point, lo, hi)
    _cabi.check_seq(_cabi.lib().qgru_norm_forward(n, torch._C._cuda_getCurrentRawStream(x2.device.index or 0)), "qgru_norm_forward")


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        x2, r2, weight = _rows(x), _rows(residual) if residual is not None else None, weight.contiguous()
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        h = torch.empty(x.shape, dtype=x.dtype, device=x.device) if residual is not None else None
        rstd = torch.empty(x2.shape[0], dtype=torch.float32, device=x.device)
        _call(x2, weight, r2, eps, h, y=y, rstd=rstd)
        ctx.save_for_backward(h if h is not None else x, weight, rstd)
        ctx.has_residual = residual is not None
        ctx.set_materialize_grads(False)
        return y if h is None else (y, h)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh=None):
        h, weight, rstd = ctx.saved_tensors
        if dy is None:                       # only the stream goes on
            return dh, None, dh if ctx.has_residual else None, None
        h2, dy2, dh2 = _rows(h), _rows(dy), _rows(dh) if dh is not None else None
        dev, (rows, cols) = h.device, h2.shape
        weight, rstd = weight.contiguous(), rstd.contiguous()
        dx = torch.empty(h.shape, dtype=h.dtype, device=dev)
        dw = torch.empty_like(weight) if ctx.needs_input_grad[1] else None
        L = _cabi.lib()
        n = _cabi.Norm(dev.index or 0, h.dtype == torch.bfloat16, weight.dtype == torch.bfloat16, cols, rows, 0.0, weight=weight.data_ptr(), rstd=rstd.data_ptr())
        bytes_ = L.qgru_norm_workspace(dev.index or 0, rows, cols) if dw is not None else 0
        ws = torch.empty(bytes_, dtype=torch.uint8, device=dev) if bytes_ else None
        _cabi.check_seq(L.qgru_norm_backward(n, h2.data_ptr(), h2.stride(0), dy2.data_ptr(), dy2.stride(0), dh2.data_ptr() if dh2 is not None else None,
                                             dh2.stride(0) if dh2 is not None else 0, dx.data_ptr(), cols, dw.data_ptr() if dw is not None else None,
                                             ws.data_ptr() if ws is not None else None, bytes_, torch._C._cuda_getCurrentRawStream(dev.index or 0)),
                        "qgru_norm_backward")
        return dx, dw, dx if ctx.has_residual else None, None


def rms_norm(x, weight, residual=None, eps=1e-6):
    """x [..., D], weight [D], residual like x or None.  Returns y, or with a residual (y, h): h = x + residual, rounded to
    their type, is the stream that goes on to the next addition, and y is the norm of what is stored."""
    _checked(x, weight, residual)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (residual is not None and residual.requires_grad)):
        return _RMSNorm.apply(x, weight, residual, eps)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    h = torch.empty(x.shape, dtype=x.dtype, device=x.device) if residual is not None else None
    _call(_rows(x), weight.contiguous(), _rows(residual) if residual is not None else None, eps, h, y=y)
    return y if h is None else (y, h)


@torch.no_grad()
def rms_norm_q8(x, weight, residual=None, eps=1e-6, scale=None, zero_point=0, bits=8, unsigned=False):
    """The norm's output in 8 bits, without a gradient.

    With ``scale=None`` every row has a scale of its own: returns (q int8, scales [...] float32[, h]) with q * scale the
    norm, |q| <= 127 (a row of zeros: 0 and 0; a row with infinities or NaN: 0 and NaN).  With a scale (and zero point, width
    and sign, as the input operator of a calibrated layer has them) returns (q[, h]), q = clamp(round(y / scale) + zero_point)
    in int8, or uint8 where ``unsigned``.  Halves round to even."""
    _checked(x, weight, residual)
    given = None
    if scale is not None:
        if not scale > 0 or not 1 <= bits <= 8:
            raise ValueError(f"scale must be positive and bits between 1 and 8, got {scale} and {bits}")
        lo, hi = (0, (1 << bits) - 1) if unsigned else (-(1 << bits - 1), (1 << bits - 1) - 1)
        if not -1 << 24 < zero_point < 1 << 24:
            raise ValueError(f"zero_point {zero_point} is out of range")
        given = (float(scale), int(zero_point), lo, hi)
    q = torch.empty(x.shape, dtype=torch.uint8 if given and unsigned else torch.int8, device=x.device)
    h = torch.empty(x.shape, dtype=x.dtype, device=x.device) if residual is not None else None
    scales = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device) if given is None else None
    _call(_rows(x), weight.contiguous(), _rows(residual) if residual is not None else None, eps, h, q8=q, scales=scales, given=given)
    return (q, *(() if scales is None else (scales,)), *(() if h is None else (h,))) if scales is not None or h is not None else q
