"""Linear attention with a decay for each head: a recurrent layer like the GRU, with the state carried by the caller, but linear
in its state and so parallel over time (no counterpart in the reference).

For every sequence and head, with the state S [Dk, Dv]

    S_t = exp(log_decay_t) S_{t-1} + k_t^T v_t,    out_t = scale * q_t S_t

``linear_attention``       whole sequences (prompts, training); differentiable
``linear_attention_step``  one token of every sequence, the state updated in place (serving)
``LinearAttention``        a layer around them: norm with the residual's addition, projections, a gate for the decays
``synchronize``            waits, and raises what went wrong inside a kernel

Tensors are [T, B, heads, D] as the GRU's are [T, B, H] ([B, T, heads, D] with ``batch_first``) with any strides whose last
is 1, float32 or bfloat16; states are float32.  Arguments are checked, memory is allocated and the library is called in
csrc/qgru_seq_torch.cc.  Everything runs on the current stream of the tensors' device, waits for nothing and may be captured into a
graph; where a backward pass is, no graph of the same leaves made on the default stream may still live (of q, k, v, log_decay and
initial_state themselves it is refused).  Gradients are of the first order and backward; inputs with a forward-mode tangent are refused.
"""
import math

import torch
from torch import nn

from . import _cabi
from .norm import rms_norm


def linear_attention(q, k, v, log_decay, initial_state=None, lengths=None, scale=None, batch_first=False):
    """q, k [T, B, Hk, Dk], v [T, B, H, Dv] (H a multiple of Hk: heads share q and k in groups of neighbours), log_decay
    [T, B, H], or [H] for decays that stay the same, float32 or the type of q, at most 0; head sizes up to 256.
    initial_state [B, H, Dk, Dv] float32 (zeros without one).  lengths [B] int32 on the device: sequence b ends after
    lengths[b] tokens (clamped to 0 .. T); what lies behind does not count, its outputs and gradients are zeros.  scale: 1 / sqrt(Dk)
    without one.  An infinity or NaN of a token reaches no earlier output; what it reaches is infinite or NaN.  Returns (out like v, the states after the last tokens [B, H, Dk, Dv] float32)."""
    return (_cabi._seq or _cabi.seq()).linear_attention(q, k, v, log_decay, initial_state, lengths, scale, batch_first)


def linear_attention_step(q, k, v, log_decay, state, scale=None):
    """One token of every sequence: q, k [B, Hk, Dk], v [B, H, Dv], log_decay [B, H] or [H].  state [B, H, Dk, Dv] float32, a
    head's state dense, is updated in place.  Returns out [B, H, Dv].  No gradient."""
    return (_cabi._seq or _cabi.seq()).linear_attention_step(q, k, v, log_decay, state, scale)


def synchronize(device=None):
    """Waits for the work on the current stream of `device` and raises what went wrong inside a kernel of these operators there (a bounded
    wait that ran out: results are unfinished), replays of captured graphs included.  Without it the next call on the device raises it."""
    device = torch.device("cuda" if device is None else device)
    stream = torch.cuda.current_stream(device)
    stream.synchronize()
    status = _cabi.lib().qgru_seq_check(stream.device_index)
    if status != _cabi.QGRU_OK:
        raise _cabi.QgruError(status, "synchronize", _cabi.lib().qgru_seq_last_error().decode())


class LinearAttention(nn.Module):
    """A layer of a stack, [T, B, input_size] to the same ([B, T, input_size] with ``batch_first``):

        y, stream = rms_norm(x, residual);  q, k, v, gate = projections of y
        o, state = linear_attention(q, k, v, logsigmoid(gate));  out = projection of rms_norm(o) per head

    ``forward(x, residual=None, state=None, lengths=None)`` returns (out, stream, state): the next layer takes out as its x and
    stream as its residual.  ``step`` does the same for one token [B, input_size] and updates the state in place."""

    def __init__(self, input_size, num_heads, key_size=64, value_size=64, num_key_heads=None, batch_first=False, eps=1e-6):
        super().__init__()
        num_key_heads = num_heads if num_key_heads is None else num_key_heads
        if min(input_size, num_heads, num_key_heads, key_size, value_size) < 1:
            raise ValueError("sizes and numbers of heads must be positive")
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
