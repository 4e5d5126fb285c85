"""Root-mean-square norm with the residual's addition, its gradient and its 8-bit output against 64 bits."""
import importlib

import pytest
import torch

from __graft_entry__ import PKG_NAME
from tests import seq_reference as ref

norm = importlib.import_module(PKG_NAME + ".norm")
pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
F = 2.0 ** -24
SHAPES = [(1, 1), (1, 512), (3, 7), (5, 321), (9, 1024), (4, 1032), (2, 4096), (3, 4100), (2, 8192), (2, 16384), (300, 96), (2000, 40)]


def make(dev, rows, cols, dtype, wtype=None, seed=0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(rows, cols, generator=gen, device=dev).to(dtype)
    r = (3 * torch.randn(rows, cols, generator=gen, device=dev)).to(dtype)
    w = (1 + 0.3 * torch.randn(cols, generator=gen, device=dev)).to(wtype or dtype)
    return x, r, w


def within(got, want, bound, name=""):
    off = (got.double() - want).abs() / (bound + 1e-300)
    assert off.max() <= 1, f"{name}: {off.max():.2f} times the bound"


# fp32 inside: the mean of squares is a sum of `cols` positive terms, whose relative error halves in the root; a few roundings more
def inner(cols):
    return (cols / 2 + 8) * F


@pytest.mark.parametrize("types", [(BF, BF), (BF, F32), (F32, F32), (F32, BF)], ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("with_residual", [False, True])
def test_norm_and_gradient(shape, types, with_residual, cuda_device):
    x, r, w = make(cuda_device, *shape, *types)
    u, uw = ref.U[types[0]], ref.U[types[1]]
    leaves = [t.requires_grad_() for t in ((x, w, r) if with_residual else (x, w))]
    dy, dh = torch.randn_like(x), torch.randn_like(x) if with_residual else None
    if with_residual:
        y, h = norm.rms_norm(x, w, r, 1e-5)
        grads = torch.autograd.grad((y, h), leaves, (dy, dh))
    else:
        y = norm.rms_norm(x, w, eps=1e-5)
        grads = torch.autograd.grad(y, leaves, dy)
    want = ref.norm(x.detach(), w.detach(), r.detach() if with_residual else None, 1e-5, dy, dh)
    if with_residual:
        assert torch.equal(h, want["h"]) and torch.equal(grads[0], grads[2])
    e = inner(shape[1])
    within(y, want["y"], (u + e) * want["y"].abs(), "y")
    within(grads[0], want["dx"], u * want["dx"].abs() + 4 * e * want["dx_size"], "dx")
    within(grads[1], want["dw"], uw * want["dw"].abs() + (e + (shape[0] + 8) * F) * want["dw_size"], "dw")
    with torch.no_grad():
        again = norm.rms_norm(x, w, r, 1e-5)[0] if with_residual else norm.rms_norm(x, w, eps=1e-5)
    assert torch.equal(again, y)


@pytest.mark.parametrize("types", [(BF, BF), (BF, F32), (F32, F32), (F32, BF)], ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("with_residual", [False, True])
def test_eight_bits_with_a_scale_for_each_row(shape, types, with_residual, cuda_device):
    x, r, w = make(cuda_device, *shape, *types)
    got = norm.rms_norm_q8(x, w, r if with_residual else None)
    want = ref.norm(x, w, r if with_residual else None)
    hw = want["h"].double() * w.double()
    top = hw.abs().amax(-1, keepdim=True)
    assert got[0].dtype == torch.int8 and torch.equal(got[0].double(), torch.round(hw * 127 / top))
    within(got[1], want["y"].abs().amax(-1) / 127, (inner(shape[1]) + 4 * F) * want["y"].abs().amax(-1) / 127, "scale")
    if with_residual:
        assert torch.equal(got[2], want["h"])


def test_halves_go_to_even(cuda_device):
    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -126.5, 3.0]], device=cuda_device)
    for t in (BF, F32):
        q, s = norm.rms_norm_q8(x.to(t), torch.ones(8, device=cuda_device, dtype=t))
        assert q[0].tolist() == [127, 0, 2, 2, 0, -2, -126, 3]


def test_rows_of_nothing_and_of_too_much(cuda_device):
    w = torch.ones(64, device=cuda_device)
    x = torch.randn(5, 64, device=cuda_device)
    x[0], x[1, 3], x[2, 4], x[4] = 0.0, float("nan"), float("inf"), x[4] * 1e-37
    q, s = norm.rms_norm_q8(x, w)
    assert (q[:3] == 0).all() and s[0] == 0 and s[1].isnan() and s[2].isnan()
    assert torch.equal(q[4].double(), torch.round(x[4].double() * 127 / x[4].double().abs().max()))
    y = norm.rms_norm(x, w)
    assert (y[0] == 0).all() and y[1].isnan().all() and torch.isfinite(y[3:]).all()


@pytest.mark.parametrize("given", [dict(scale=0.031), dict(scale=0.02, zero_point=-7), dict(scale=0.05, zero_point=100, unsigned=True), dict(scale=0.4, bits=5)], ids=str)
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_eight_bits_with_a_given_scale(given, dtype, cuda_device):
    x, r, w = make(cuda_device, 50, 161, dtype)
    q, h = norm.rms_norm_q8(x, w, r, **given)
    want = ref.norm(x, w, r)
    assert torch.equal(h, want["h"])
    bits, unsigned = given.get("bits", 8), given.get("unsigned", False)
    lo, hi = (0, 2 ** bits - 1) if unsigned else (-2 ** (bits - 1), 2 ** (bits - 1) - 1)
    assert q.dtype == (torch.uint8 if unsigned else torch.int8)
    t = want["y"] / float(torch.tensor(given["scale"]))
    exact = (torch.round(t) + given.get("zero_point", 0)).clamp(lo, hi)
    near = ((t - t.floor()) - 0.5).abs() <= (inner(161) + 4 * F) * t.abs()       # fp32 may take either side there
    assert (near | (q.double() == exact)).all() and ((q.double() - exact).abs() <= 1).all() and near.float().mean() < 1e-3


def test_strides_and_leading_dimensions(cuda_device):
    x = torch.randn(6, 5, 3, 80, device=cuda_device).transpose(0, 1)
    w = torch.ones(64, device=cuda_device)
    for t in (x[..., :64], x[..., 1:65], x[:, :, 0, 16:]):
        assert torch.equal(norm.rms_norm(t, w), norm.rms_norm(t.contiguous(), w))
        a, b = norm.rms_norm_q8(t, w), norm.rms_norm_q8(t.contiguous(), w)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and a[1].shape == t.shape[:-1]
    t = x[..., 1:65].detach().requires_grad_()
    w.requires_grad_()
    dy = torch.randn(5, 6, 3, 128, device=cuda_device)[..., ::2]
    got = torch.autograd.grad(norm.rms_norm(t, w), (t, w), dy)
    dense = t.detach().contiguous().requires_grad_()
    want = torch.autograd.grad(norm.rms_norm(dense, w), (dense, w), dy.contiguous())
    for a, b in zip(got, want):          # (vectors or single elements: sums of another order)
        assert (a - b).abs().max() <= 90 * 16 * F * b.abs().max()
    empty = torch.empty(0, 64, device=cuda_device, requires_grad=True)
    g = torch.autograd.grad(norm.rms_norm(empty, w).sum(), (empty, w))
    assert g[0].shape == (0, 64) and (g[1] == 0).all()


def test_one_output_alone_gets_a_gradient(cuda_device):
    x, r, w = make(cuda_device, 10, 64, F32)
    x.requires_grad_(), r.requires_grad_(), w.requires_grad_()
    y, h = norm.rms_norm(x, w, r)
    gx, gr = torch.autograd.grad(h.sum(), (x, r), retain_graph=True)
    assert (gx == 1).all() and (gr == 1).all()
    a = torch.autograd.grad(y.square().sum(), (x, w), retain_graph=True)
    y2, _ = norm.rms_norm(x, w, r)
    b = torch.autograd.grad((y2.square().sum()), (x, w))
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_gradient_against_differences(cuda_device):
    x, r, w = make(cuda_device, 6, 50, F32)
    x.requires_grad_(), w.requires_grad_()
    a = torch.randn(6, 50, device=cuda_device)
    grads = torch.autograd.grad(norm.rms_norm(x, w), (x, w), a)
    for i, t in enumerate((x, w)):
        d = torch.randn_like(t)
        with torch.no_grad():
            f = [(norm.rms_norm(x + e * d if i == 0 else x, w + e * d if i == 1 else w).double() * a).sum() for e in (1e-2, -1e-2)]
        # 300 terms of size about 3 rounded in fp32 over 2e-2, and the cubic term of the quotient, below 1e-4 of the terms' norm
        tol = 300 * 3 * F / 2e-2 + 1e-3 * grads[i].double().norm() * d.double().norm() / 10
        assert abs((f[0] - f[1]) / 2e-2 - (grads[i].double() * d).sum()) <= tol


def test_captured_and_on_other_streams(cuda_device):
    x, r, w = make(cuda_device, 400, 512, BF)
    want = norm.rms_norm_q8(x, w, r)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        got = norm.rms_norm_q8(x, w, r)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = norm.rms_norm_q8(x, w, r)
    x.mul_(-2.0)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(norm.rms_norm_q8(x, w, r), got))


def test_offsets_beyond_32_bits(cuda_device):
    """2.2e9 elements: the last rows as they are alone."""
    x = torch.empty(270000, 8192, dtype=BF, device=cuda_device).normal_().requires_grad_()
    w = torch.ones(8192, dtype=BF, device=cuda_device)
    y = norm.rms_norm(x, w)
    dx, = torch.autograd.grad(y, x, x.detach())
    q, s = norm.rms_norm_q8(x.detach(), w)
    part = x.detach()[-3:].contiguous().requires_grad_()
    y1 = norm.rms_norm(part, w)
    dx1, = torch.autograd.grad(y1, part, part.detach())
    q1, s1 = norm.rms_norm_q8(part.detach(), w)
    assert torch.equal(y[-3:], y1) and torch.equal(dx[-3:], dx1) and torch.equal(q[-3:], q1) and torch.equal(s[-3:], s1)


def test_a_captured_training_step(cuda_device):
    x, r, w = make(cuda_device, 300, 512, BF)
    leaves = [t.requires_grad_() for t in (x, w, r)]
    dy, dh = torch.randn_like(x), torch.randn_like(x)

    def run():
        y, h = norm.rms_norm(x, w, r)
        return [y.detach(), *torch.autograd.grad((y, h), leaves, (dy, dh))]

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = run()
    with torch.no_grad():
        x.mul_(-0.5)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(run(), got))


def test_a_second_derivative_is_refused(cuda_device):
    x, r, w = make(cuda_device, 3, 40, F32)
    x.requires_grad_()
    dx, = torch.autograd.grad(norm.rms_norm(x, w).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        dx.sum().backward()


def test_before_a_quantized_layer(cuda_device):
    """The norm's output in the integers that a calibrated QuantGRU takes, with the scale of its own input operator."""
    import numpy as np
    from tests.cases import OP
    QuantGRU = importlib.import_module(PKG_NAME + ".quant_gru").QuantGRU
    torch.manual_seed(0)
    module = QuantGRU(48, 64, use_quantization=True, quant_storage_dtype="int32").to(cuda_device).eval()
    module.set_all_bitwidth(8, True)
    x, r = torch.randn(30, 4, 48, device=cuda_device), torch.randn(30, 4, 48, device=cuda_device)
    w = torch.ones(48, device=cuda_device)
    y, _ = norm.rms_norm(x, w, r)
    module.calibrating = True
    module(y)
    module.calibrating = False
    module.finalize_calibration()
    op = module.quant_params.c.op[OP["x"]]
    scale = importlib.import_module(PKG_NAME + ".gru_ops").decode_effective_scale(op.scale, False)
    q, h = norm.rms_norm_q8(x, w, r, scale=scale, zero_point=op.zero_point, bits=op.bits, unsigned=bool(op.is_unsigned))
    out, hn = module.forward_quantized(q)
    want, want_hn = module(y)
    meta = module._dirs[0].handle.h_quant_meta()
    back = (out.float() - meta[1]) * meta[0]
    # the same integers but for values at a border of the rounding, which fp32 may take either way
    t = y.double() / scale
    if not ((t - t.floor()) - 0.5).abs().min() < 1e-4:
        assert np.array_equal(back.cpu().numpy(), want.cpu().numpy())
    assert (back - want).abs().max() <= 4 * meta[0]


def test_refusals(cuda_device):
    x, r, w = make(cuda_device, 4, 32, BF)
    for bad in (lambda: norm.rms_norm(x.cpu(), w), lambda: norm.rms_norm(x.half(), w), lambda: norm.rms_norm(x, w[:31]), lambda: norm.rms_norm(x, w.half()),
                lambda: norm.rms_norm(x, w, r.float()), lambda: norm.rms_norm(x, w, r[:3]), lambda: norm.rms_norm_q8(x, w, scale=0.0),
                lambda: norm.rms_norm_q8(x, w, scale=0.1, bits=9), lambda: norm.rms_norm_q8(x, w, scale=0.1, zero_point=1 << 25), lambda: norm.rms_norm(x[:, :0], w[:0])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="columns"):
        norm.rms_norm(torch.ones(1, 16385, device=cuda_device), torch.ones(16385, device=cuda_device))


def test_a_capture_beside_a_living_graph_is_refused(cuda_device):
    x, r, w = make(cuda_device, 30, 512, BF)
    leaves = [t.requires_grad_() for t in (x, w, r)]
    for only in range(3):
        use = [t if i == only else t.detach() for i, t in enumerate(leaves)]
        alive = norm.rms_norm(*use)                             # on the default stream
        side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            something = torch.zeros(8, device=cuda_device)
            with pytest.raises(RuntimeError, match="still lives"):
                norm.rms_norm(*use)
        graph.replay()
        torch.cuda.synchronize()
        assert not something.any()
        del alive, graph


def test_eight_bits_do_not_cut_a_stream_that_has_a_gradient(cuda_device):
    x, r, w = make(cuda_device, 3, 512, BF)
    for a, b in ((x.detach().requires_grad_(), r), (x, r.detach().requires_grad_())):
        with pytest.raises(RuntimeError, match="no gradient"):
            norm.rms_norm_q8(a, w, b)
        with torch.no_grad():
            norm.rms_norm_q8(a, w, b)
    norm.rms_norm_q8(x, w.detach().requires_grad_(), r)         # a layer's weight alone has no part in the stream
