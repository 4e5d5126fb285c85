"""Linear attention with a decay for each head: a recurrent layer like the GRU, with the state carried by the caller, but linear
in its state and so parallel over time (no counterpart in the reference).

For every sequence and head, with the state S [Dk, Dv]

    S_t = exp(log_decay_t) S_{t-1} + k_t^T v_t,    out_t = scale * q_t S_t

``linear_attention``       whole sequences (prompts, training); differentiable
``linear_attention_step``  one token of every sequence, the state updated in place (serving)
``LinearAttention``        a layer around them: norm with the residual's addition, projections, a gate for the decays

Tensors are [T, B, heads, D] as the GRU's are [T, B, H] ([B, T, heads, D] with ``batch_first``) with any strides whose last
is 1, float32 or bfloat16; states are float32.  Everything runs on the current stream of the tensors' device, waits for nothing and
may be captured into a graph.
"""
import ctypes as C
import math

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _cabi
from .norm import rms_norm

_TYPES = (torch.float32, torch.bfloat16)
_NONE = (None, 0, 0, 0)
_BLANK = (None,) * 7 + (0, 0) + (_NONE,) * 10


def _tensor(t, name, dtype, device, shape):
    if not isinstance(t, torch.Tensor) or t.device != device or t.dtype != dtype:
        raise ValueError(f"{name} must be a {dtype} tensor on {device}")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {list(shape)}, got {list(t.shape)}")
    return t


def _readable(t):
    """t, or a dense copy where its last stride is not 1 or its rows could be fetched in 16-byte pieces but for where they lie."""
    if t.numel() == 0:
        return t
    per = 16 // t.element_size()
    s = t.stride()
    if s[-1] == 1 and (t.shape[-1] % per or not (t.data_ptr() % 16 or any(x % per for x in s[:-1]))):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _check(q, k, v, log_decay, lead):
    """Shapes and types; the log decay as [*lead, H]."""
    for name, t in (("q", q), ("k", k), ("v", v)):
        if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype not in _TYPES:
            raise ValueError(f"{name} must be a CUDA tensor of float32 or bfloat16")
        if t.dim() != lead + 2:
            raise ValueError(f"{name} must have {lead + 2} dimensions, got shape {list(t.shape)}")
    _tensor(k, "k", q.dtype, q.device, q.shape)
    if v.dtype != q.dtype or v.device != q.device or v.shape[:lead] != q.shape[:lead]:
        raise ValueError(f"v must be a {q.dtype} tensor on {q.device} that begins with {list(q.shape[:lead])}, got {list(v.shape)}")
    H, Hk = v.shape[lead], q.shape[lead]
    if H < 1 or Hk < 1 or q.shape[-1] < 1 or v.shape[-1] < 1:
        raise ValueError("heads and head sizes must be positive")
    if H % Hk:
        raise ValueError(f"{H} heads cannot share {Hk} heads of q and k")
    if not isinstance(log_decay, torch.Tensor) or log_decay.device != q.device or log_decay.dtype not in (torch.float32, q.dtype):
        raise ValueError(f"log_decay must be a float32 or {q.dtype} tensor on {q.device}")
    if log_decay.shape == (H,):
        log_decay = log_decay.expand(*q.shape[:lead], H)
    elif log_decay.shape != v.shape[:lead + 1]:
        raise ValueError(f"log_decay must have shape {[H]} or {list(v.shape[:lead + 1])}, got {list(log_decay.shape)}")
    return log_decay


def _head(dims, dev, q, decay, scale, keep=False):
    T, B, H, Hk, Dk, Dv = dims
    return _cabi.Attention(dev, T, B, H, Hk, Dk, Dv, q.dtype == torch.bfloat16, decay.dtype == torch.bfloat16, keep, scale, *_BLANK)


def _place(t, batch_first):
    s = t.stride()
    ts, bs = (s[1], s[0]) if batch_first else (s[0], s[1])
    return (t.data_ptr(), ts, bs, s[2])


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _block(nbytes, device):
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _forward(q, k, v, decay, state0, lengths, scale, batch_first, keep):
    """-> out, state, states (what the backward reads, with `keep`)."""
    q, k, v = _readable(q), _readable(k), _readable(v)
    t_dim, b_dim = (1, 0) if batch_first else (0, 1)
    dims = (q.shape[t_dim], q.shape[b_dim], v.shape[2], q.shape[2], q.shape[3], v.shape[3])
    T, B, H, _, Dk, Dv = dims
    device, dev, L = q.device, q.device.index or 0, _cabi.lib()
    a = _head(dims, dev, q, decay, scale, keep)
    a.q, a.k, a.v, a.decay = (_place(x, batch_first) for x in (q, k, v, decay))
    sizes = [C.c_size_t() for _ in range(3)]
    _cabi.check_seq(L.qgru_attention_sizes(a, *sizes), "qgru_attention_sizes")
    states, ws = _block(sizes[0].value, device), _block(sizes[1].value, device)
    out = torch.empty(v.shape, dtype=v.dtype, device=device)
    state = torch.empty((B, H, Dk, Dv), dtype=torch.float32, device=device)
    a.lengths, a.state0, a.state, a.states, a.workspace = _ptr(lengths), _ptr(state0), state.data_ptr(), _ptr(states), _ptr(ws)
    a.states_bytes, a.workspace_bytes = sizes[0].value, sizes[1].value
    a.out = _place(out, batch_first)
    _cabi.check_seq(L.qgru_attention_forward(a, torch._C._cuda_getCurrentRawStream(dev)), "qgru_attention_forward")
    return out, state, states


class _LinearAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, decay, state0, lengths, scale, batch_first):
        out, state, states = _forward(q, k, v, decay, state0, lengths, scale, batch_first, True)
        ctx.save_for_backward(q, k, v, decay, lengths, states)
        ctx.scale, ctx.batch_first, ctx.has_state = scale, batch_first, state0 is not None
        ctx.states_as = None if states is None else (states.shape, states.device)
        ctx.set_materialize_grads(False)
        return out, state

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dstate):
        q, k, v, decay, lengths, states = ctx.saved_tensors
        if states is not None:
            if (states.shape, states.device) != ctx.states_as or states.dtype != torch.uint8:
                raise RuntimeError("a saved-tensor hook has returned another type, shape or device than it was given")
            if not states.is_contiguous() or states.data_ptr() % 256:      # (a hook's copy: the library reads it in vectors)
                states = states.clone(memory_format=torch.contiguous_format)
        batch_first = ctx.batch_first
        t_dim, b_dim = (1, 0) if batch_first else (0, 1)
        q, k, v = _readable(q), _readable(k), _readable(v)
        dims = (q.shape[t_dim], q.shape[b_dim], v.shape[2], q.shape[2], q.shape[3], v.shape[3])
        device, dev, L = q.device, q.device.index or 0, _cabi.lib()
        dout = torch.zeros(v.shape, dtype=v.dtype, device=device) if dout is None else _readable(dout)
        dstate = dstate.contiguous() if dstate is not None else None
        a = _head(dims, dev, q, decay, ctx.scale, True)
        for name, t in (("q", q), ("k", k), ("v", v), ("decay", decay), ("dout", dout)):
            setattr(a, name, _place(t, batch_first))
        sizes = [C.c_size_t() for _ in range(3)]
        _cabi.check_seq(L.qgru_attention_sizes(a, *sizes), "qgru_attention_sizes")
        ws = _block(sizes[2].value, device)
        dq, dk, dv, dg = (torch.empty(t.shape, dtype=t.dtype, device=device) for t in (q, k, v, decay))
        dstate0 = torch.empty((dims[1], dims[2], dims[4], dims[5]), dtype=torch.float32, device=device) if ctx.has_state and ctx.needs_input_grad[4] else None
        a.lengths, a.dstate, a.dstate0, a.states, a.workspace = _ptr(lengths), _ptr(dstate), _ptr(dstate0), _ptr(states), _ptr(ws)
        a.states_bytes, a.workspace_bytes = sizes[0].value, sizes[2].value
        for name, t in (("dq", dq), ("dk", dk), ("dv", dv), ("ddecay", dg)):
            setattr(a, name, _place(t, batch_first))
        _cabi.check_seq(L.qgru_attention_backward(a, torch._C._cuda_getCurrentRawStream(dev)), "qgru_attention_backward")
        return dq, dk, dv, dg, dstate0, None, None, None


def linear_attention(q, k, v, log_decay, initial_state=None, lengths=None, scale=None, batch_first=False):
    """q, k [T, B, Hk, Dk], v [T, B, H, Dv] (H a multiple of Hk: heads share q and k in groups of neighbours), log_decay
    [T, B, H], or [H] for decays that stay the same, float32 or the type of q, at most 0; head sizes up to 256.
    initial_state [B, H, Dk, Dv] float32 (zeros without one).  lengths [B] int32 on the device: sequence b ends after
    lengths[b] tokens (clamped to 0 .. T); what lies behind is not read, its outputs and gradients are zeros.  scale: 1 / sqrt(Dk)
    without one.  Returns (out like v, the states after the last tokens [B, H, Dk, Dv] float32)."""
    log_decay = _check(q, k, v, log_decay, 2)
    B = q.shape[0 if batch_first else 1]
    if initial_state is not None:
        initial_state = _tensor(initial_state, "initial_state", torch.float32, q.device, (B, v.shape[2], q.shape[3], v.shape[3])).contiguous()
    if lengths is not None:
        lengths = _tensor(lengths, "lengths", torch.int32, q.device, (B,)).contiguous()
    scale = q.shape[3] ** -0.5 if scale is None else float(scale)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, log_decay, initial_state)):
        return _LinearAttention.apply(q, k, v, log_decay, initial_state, lengths, scale, batch_first)
    return _forward(q, k, v, log_decay, initial_state, lengths, scale, batch_first, False)[:2]


def linear_attention_step(q, k, v, log_decay, state, scale=None):
    """One token of every sequence: q, k [B, Hk, Dk], v [B, H, Dv], log_decay [B, H] or [H].  state [B, H, Dk, Dv] float32, a
    head's state dense, is updated in place.  Returns out [B, H, Dv].  No gradient."""
    log_decay = _check(q, k, v, log_decay, 1)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or log_decay.requires_grad or
                                    (isinstance(state, torch.Tensor) and state.requires_grad)):
        raise RuntimeError("linear_attention_step has no gradient: call it under torch.no_grad(), or linear_attention with T = 1")
    (B, Hk, Dk), (_, H, Dv) = q.shape, v.shape
    _tensor(state, "state", torch.float32, q.device, (B, H, Dk, Dv))
    bs, hs, ks, vs = state.stride()
    dense = (vs == 1 or Dv == 1) and (ks == Dv or Dk == 1)
    apart = (H == 1 or hs >= Dk * Dv) and (B == 1 or bs >= Dk * Dv) and (H == 1 or B == 1 or bs >= H * hs or hs >= B * bs)
    if B and not (dense and apart):
        raise ValueError(f"a head's state must be dense and the states must not overlap, got strides {list(state.stride())}")
    q, k, v = _readable(q), _readable(k), _readable(v)
    out = torch.empty((B, H, Dv), dtype=q.dtype, device=q.device)
    dev = q.device.index or 0
    a = _head((1, B, H, Hk, Dk, Dv), dev, q, log_decay, Dk ** -0.5 if scale is None else float(scale))
    a.state = state.data_ptr()
    for name, t in (("q", q), ("k", k), ("v", v), ("decay", log_decay), ("out", out)):
        setattr(a, name, (t.data_ptr(), 0, t.stride(0), t.stride(1)))
    _cabi.check_seq(_cabi.lib().qgru_attention_step(a, bs, hs, torch._C._cuda_getCurrentRawStream(dev)), "qgru_attention_step")
    torch.autograd.graph.increment_version(state)
    return out


class LinearAttention(nn.Module):
    """A layer of a stack, [T, B, input_size] to the same ([B, T, input_size] with ``batch_first``):

        y, stream = rms_norm(x, residual);  q, k, v, gate = projections of y
        o, state = linear_attention(q, k, v, logsigmoid(gate));  out = projection of rms_norm(o) per head

    ``forward(x, residual=None, state=None, lengths=None)`` returns (out, stream, state): the next layer takes out as its x and
    stream as its residual.  ``step`` does the same for one token [B, input_size] and updates the state in place."""

    def __init__(self, input_size, num_heads, key_size=64, value_size=64, num_key_heads=None, batch_first=False, eps=1e-6):
        super().__init__()
        num_key_heads = num_key_heads or num_heads
        if num_heads % num_key_heads:
            raise ValueError(f"{num_heads} heads cannot share {num_key_heads} heads of q and k")
        self.input_size, self.num_heads, self.num_key_heads = input_size, num_heads, num_key_heads
        self.key_size, self.value_size, self.batch_first, self.eps = key_size, value_size, batch_first, eps
        self.sizes = [num_key_heads * key_size, num_key_heads * key_size, num_heads * value_size, num_heads]
        self.norm_weight = nn.Parameter(torch.empty(input_size))
        self.weight_in = nn.Parameter(torch.empty(sum(self.sizes), input_size))
        self.gate_bias = nn.Parameter(torch.empty(num_heads))
        self.head_weight = nn.Parameter(torch.empty(value_size))
        self.weight_out = nn.Parameter(torch.empty(input_size, num_heads * value_size))
        self.reset_parameters()

    def reset_parameters(self):
        for w in (self.weight_in, self.weight_out):
            nn.init.uniform_(w, -1.0 / math.sqrt(w.shape[1]), 1.0 / math.sqrt(w.shape[1]))
        nn.init.ones_(self.norm_weight)
        nn.init.ones_(self.head_weight)
        with torch.no_grad():                # memories from a few tokens to about a thousand
            self.gate_bias.copy_(torch.linspace(1.0, 7.0, self.num_heads))

    def _project(self, x, residual):
        if x.shape[-1] != self.input_size:
            raise ValueError(f"input must have {self.input_size} features, got {list(x.shape)}")
        y, stream = (rms_norm(x, self.norm_weight, eps=self.eps), x) if residual is None else rms_norm(x, self.norm_weight, residual, self.eps)
        q, k, v, gate = nn.functional.linear(y, self.weight_in).split(self.sizes, dim=-1)
        decay = nn.functional.logsigmoid(gate.float() + self.gate_bias)
        heads = self.num_key_heads
        return q.unflatten(-1, (heads, self.key_size)), k.unflatten(-1, (heads, self.key_size)), v.unflatten(-1, (self.num_heads, self.value_size)), decay, stream

    def _finish(self, o):
        return nn.functional.linear(rms_norm(o, self.head_weight, eps=self.eps).flatten(-2), self.weight_out)

    def forward(self, x, residual=None, state=None, lengths=None):
        if x.dim() != 3:
            raise ValueError(f"input must have three dimensions, got shape {list(x.shape)}")
        q, k, v, decay, stream = self._project(x, residual)
        o, state = linear_attention(q, k, v, decay, state, lengths, batch_first=self.batch_first)
        return self._finish(o), stream, state

    @torch.no_grad()
    def step(self, x, state, residual=None):
        if x.dim() != 2:
            raise ValueError(f"a step's input must have two dimensions, got shape {list(x.shape)}")
        q, k, v, decay, stream = self._project(x, residual)
        return self._finish(linear_attention_step(q, k, v, decay, state)), stream
