"""layer_norm on the GPU against the formula in float64: outputs, the sum, every gradient;
widths around the kernels' thread counts and odd ones, row counts from none up, a residual
of either type, extreme rows, determinism, graph capture and the pre-norm block that runs it.

Tolerances. Every element of y and of the gradients is a sum of a few terms, each with a
few fp32 roundings (eps = 2^-24), so the error is a small multiple of eps times the size of
the terms: 64 eps of the largest value in the tensor covers the two tree sums of a row
(log2 32768 = 15 additions deep each) and the final products. A result stored in bf16 adds
half a step, 2^-8 relative. A gradient summed over n rows is summed in runs of at most
max(n / CTAs, 32) rows: its error is at most that many eps of the sum of the terms'
absolute values."""
from __future__ import annotations

import pytest
import torch

from tests.parity import cuda, gen, randn

EPS32 = 2.0 ** -24
HALF_STEP = {torch.float32: EPS32, torch.bfloat16: 2.0 ** -8}


def _reference(x, w, b, r, eps, dy, ds):
    s = x if r is None else x + r
    mean = s.mean(-1, keepdim=True)
    e = s - mean
    rstd = 1 / torch.sqrt((e * e).mean(-1, keepdim=True) + eps)
    xhat = e * rstd
    y = xhat * w + b
    g = dy * w
    dx = rstd * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
    if ds is not None:
        dx = dx + ds
    rows = tuple(range(dy.dim() - 1))
    return s, y, dx, (dy * xhat).sum(rows), dy.sum(rows), (dy * xhat).abs().sum(rows), dy.abs().sum(rows), rstd


def _near(got, want, dtype, scale=None, depth=64.0, what=""):
    got, want = got.detach().double().cpu(), want.double()
    scale = want.abs().max() if scale is None else scale
    tol = depth * EPS32 * scale + (HALF_STEP[dtype] * want.abs() if dtype != torch.float32 else 0)
    bad = (got - want).abs() - tol
    assert got.shape == want.shape and bool((bad <= 0).all()), f"{what}: over by {bad.max().item():.3e}"


SHAPES = [(1, 1), (3, 2), (5, 7), (4, 63), (17, 64), (33, 65), (9, 128), (6, 250), (7, 257), (5, 512), (3, 1000),
          (2, 1024), (3, 1030), (2, 2048), (3, 2049), (2, 4100), (2, 8192), (1, 9001), (2, 16384), (1, 32768), (1, 32767)]


@pytest.mark.gpu
@pytest.mark.parametrize("n,d", SHAPES)
@pytest.mark.parametrize("xt,rt", [(torch.float32, None), (torch.bfloat16, None), (torch.bfloat16, torch.float32),
                                   (torch.bfloat16, torch.bfloat16), (torch.float32, torch.bfloat16)])
def test_layer_norm(n, d, xt, rt):
    from semambaxlinoss_b200.layer_norm import layer_norm

    dev, g = cuda(), gen(n * 40000 + d)
    x = randn((n, d), g).to(xt)
    r = None if rt is None else randn((n, d), g).to(rt)
    w, b = randn((d,), g, scale=0.3, mean=1.0).float(), randn((d,), g).float()
    dy = randn((n, d), g).to(xt)
    st = xt if r is None else torch.promote_types(xt, rt)
    ds = None if r is None else randn((n, d), g).to(st)
    leaves = [t.to(dev).requires_grad_() for t in (x, w, b)] + ([] if r is None else [r.to(dev).requires_grad_()])
    out = layer_norm(*leaves[:3], residual=None if r is None else leaves[3])
    outs = (out,) if r is None else out
    grads = torch.autograd.grad(outs, leaves, [dy.to(dev)] + ([] if r is None else [ds.to(dev)]))
    # The norm is that of the stored sum: the reference takes the sum from the kernel after checking it.
    args = [t.double() for t in (x, w, b)]
    if r is None:
        s64, r64 = args[0], None
    else:
        s64, r64 = outs[1].detach().double().cpu(), torch.zeros(n, d, dtype=torch.float64)
        _near(outs[1], x.double() + r.double(), st, what="sum")
        assert outs[1].dtype == st
    _, y, dx, dw, db, dw_abs, db_abs, rstd = _reference(s64, args[1], args[2], r64, 1e-5, dy.double(),
                                                       None if ds is None else ds.double())
    # Rounding of s - mean and of rstd: relative to the largest |s| of the row, times rstd.
    grow = (s64.abs().amax() * rstd.max()).clamp_min(1.0)
    _near(outs[0], y, xt, scale=(grow * w.abs().max() + b.abs().max()).double(), what="y")
    gs = (rstd.max() * (dy.double() * args[1]).abs().max() * grow * grow + (0 if ds is None else ds.double().abs().max()))
    _near(grads[0], dx, xt, scale=gs, what="dx")
    _near(grads[1], dw, torch.float32, scale=dw_abs + n * EPS32 + dy.double().abs().sum(0) * grow, what="dw")
    _near(grads[2], db, torch.float32, scale=db_abs, what="db")
    if r is not None:
        assert grads[3].dtype == rt
        _near(grads[3], dx, rt, scale=gs, what="dr")
    with torch.no_grad():
        again = layer_norm(*[t.detach() for t in leaves[:3]], residual=None if r is None else leaves[3].detach())
    assert torch.equal(outs[0], again if r is None else again[0])


@pytest.mark.gpu
def test_far_mean_and_flat_rows():
    """Rows far from zero keep their variance (the squares are taken about the mean), a flat
    row gives the bias alone, a row with a NaN or an infinity gives NaN there and leaves its
    neighbours as they are."""
    from semambaxlinoss_b200.layer_norm import layer_norm

    dev = cuda()
    for d in (48, 1000, 2048, 5000):
        x = torch.arange(d, dtype=torch.float64).fmod(7) + 4096.0
        rows = torch.stack([x, torch.full((d,), 3.0, dtype=torch.float64), x, x, x])
        rows[2, d // 2] = float("nan")
        rows[3, d - 1] = float("inf")
        b = torch.linspace(-1, 1, d, dtype=torch.float64)
        y = layer_norm(rows.float().to(dev), torch.ones(d, device=dev), b.float().to(dev)).double().cpu()
        want = (x - x.mean()) / torch.sqrt(x.var(correction=0) + 1e-5) + b
        # |s| rstd is 2048: the mean's own rounding, a few steps of 4096 2^-24, shows 2048 fold.
        assert (y[0] - want).abs().max() < 16 * 4096 * EPS32 / 2 + 64 * EPS32 * 4
        assert torch.equal(y[4], y[0])
        assert (y[1] - b).abs().max() <= 64 * EPS32 * 3 * 317  # rstd of a flat row: 1 / sqrt(1e-5)
        assert torch.isnan(y[2]).all() and torch.isnan(y[3]).all()


@pytest.mark.gpu
def test_many_rows_deterministic_and_no_rows():
    from semambaxlinoss_b200.layer_norm import layer_norm

    dev = cuda()
    x = torch.randn(20011, 64, device=dev)
    dy = torch.randn_like(x)

    def run():
        w, b = torch.ones(64, device=dev, requires_grad=True), torch.zeros(64, device=dev, requires_grad=True)
        return torch.autograd.grad(layer_norm(x, w, b), (w, b), dy)

    first, second = run(), run()
    assert all(torch.equal(p, q) for p, q in zip(first, second))
    xd = x.double()
    xhat = (xd - xd.mean(-1, keepdim=True)) / torch.sqrt(xd.var(-1, correction=0, keepdim=True) + 1e-5)
    # 592 CTAs of 16 rows: runs of at most 16 x 3 rows, then 32, then 19 partial sums.
    tol = (3 + 16 + 32 + 19 + 64) * EPS32 * (dy.double() * xhat).abs().sum(0).max()
    assert (first[0].double() - (dy.double() * xhat).sum(0)).abs().max() <= tol
    empty = torch.empty(0, 64, device=dev, requires_grad=True)
    w = torch.ones(64, device=dev, requires_grad=True)
    y = layer_norm(empty, w, None)
    assert y.shape == (0, 64)
    gx, gw = torch.autograd.grad(y, (empty, w), torch.empty(0, 64, device=dev))
    assert gx.shape == (0, 64) and torch.equal(gw, torch.zeros(64, device=dev))


@pytest.mark.gpu
def test_views_types_missing_parameters_and_gradients_asked_for():
    from semambaxlinoss_b200.layer_norm import layer_norm

    dev = cuda()
    base = torch.randn(6, 5, 130, device=dev)
    x = base[..., 1:129].transpose(0, 1)  # neither contiguous nor aligned
    want = torch.nn.functional.layer_norm(x.double(), (128,))
    assert (layer_norm(x, None).double() - want).abs().max() < 64 * EPS32 * 8
    y = layer_norm(x, None, out_dtype=torch.bfloat16)
    assert y.dtype == torch.bfloat16 and (y.double() - want).abs().max() <= 2.0 ** -8 * want.abs().max()
    # Unaligned rows: the same values as aligned ones.
    flat = torch.randn(4 * 64 + 1, device=dev)
    assert torch.equal(layer_norm(flat[1:].view(4, 64), None), layer_norm(flat[1:].view(4, 64).clone(), None)) or (
        layer_norm(flat[1:].view(4, 64), None) - layer_norm(flat[1:].view(4, 64).clone(), None)).abs().max() < 64 * EPS32 * 8
    # Only the sum's gradient, only the weight's, parameters in bf16.
    r = torch.randn(3, 64, device=dev, requires_grad=True)
    w = torch.ones(64, device=dev, dtype=torch.bfloat16, requires_grad=True)
    y, s = layer_norm(torch.randn(3, 64, device=dev), w, None, residual=r)
    g = torch.randn_like(s)
    (dr,) = torch.autograd.grad(s, r, g, retain_graph=True)
    assert torch.equal(dr, g)
    (dw,) = torch.autograd.grad(y, w, g)
    assert dw.dtype == torch.bfloat16
    with pytest.raises(RuntimeError):
        torch.autograd.grad(torch.autograd.grad(layer_norm(r, None).sum(), r, create_graph=True)[0].sum(), r)


@pytest.mark.gpu
def test_gradients_against_differences():
    """The operator's own outputs, moved along one direction of every operand by 2^-7: the slope
    to about 4 (2^-7)^2 of the terms' size, and the outputs' rounding, 64 2^-24, over the step."""
    from semambaxlinoss_b200.layer_norm import layer_norm

    dev, g = cuda(), gen(77)
    t = [randn(s, g).float().to(dev) for s in ((9, 130), (130,), (130,), (9, 130))]
    move = [randn(u.shape, g, scale=0.3).float().to(dev) for u in t]
    cy, cs = (randn((9, 130), g).float().to(dev) for _ in range(2))

    def value(x, w, b, r):
        y, s = layer_norm(x, w, b, residual=r)
        return (y.double() * cy).sum() + (s.double() * cs).sum(), y, s

    leaves = [u.clone().requires_grad_() for u in t]
    _, y, s = value(*leaves)
    grads = torch.autograd.grad((y, s), leaves, (cy, cs))
    slope = sum((p.double() * m.double()).sum() for p, m in zip(grads, move))
    size = sum((p.double() * m.double()).abs().sum() for p, m in zip(grads, move))
    h = 2.0 ** -7
    up, down = (value(*[u + k * h * m for u, m in zip(t, move)])[0] for k in (1, -1))
    noise = 64 * EPS32 / h * ((y.double() * cy).abs().sum() + (s.double() * cs).abs().sum())
    assert ((up - down) / (2 * h) - slope).abs() <= 4 * h * h * size + noise


@pytest.mark.gpu
def test_other_stream_and_captured_graph():
    from semambaxlinoss_b200.layer_norm import layer_norm

    dev = cuda()
    x, r = torch.randn(300, 384, device=dev), torch.randn(300, 384, device=dev)
    w, b = torch.randn(384, device=dev, requires_grad=True), torch.randn(384, device=dev, requires_grad=True)
    dy = torch.randn_like(x)

    def run():
        y, s = layer_norm(x, w, b, residual=r)
        return (y.detach(), s.detach()) + torch.autograd.grad(y, (w, b), dy)

    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    del got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    x.copy_(torch.randn_like(x))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(run(), out))


def test_refusals():
    """Checks that run before any device access."""
    from semambaxlinoss_b200 import _lib
    from semambaxlinoss_b200.layer_norm import LayerNorm, layer_norm

    with pytest.raises(RuntimeError):
        layer_norm(torch.randn(2, 8), None)
    with pytest.raises(RuntimeError):
        LayerNorm(8)(torch.randn(2, 8))
    import ctypes

    lib = _lib.load()

    def status(entry, **fields):
        a = _lib.new_args(_lib.SemxLayerNormArgs)
        a.n, a.d, a.eps = 2, 8, 1e-5
        for k, v in fields.items():
            setattr(a, k, v)
        return getattr(lib, entry)(ctypes.byref(a), None)

    assert status("semx_layer_norm_fwd", struct_size=8) == _lib.SEMX_ERR_ABI
    assert status("semx_layer_norm_fwd") == _lib.SEMX_ERR_NULL
    assert status("semx_layer_norm_fwd", d=0) == _lib.SEMX_ERR_SHAPE
    assert status("semx_layer_norm_fwd", d=32769) == _lib.SEMX_ERR_UNSUPPORTED
    assert status("semx_layer_norm_fwd", n=-1) == _lib.SEMX_ERR_SHAPE
    assert status("semx_layer_norm_fwd", n=2 ** 62) == _lib.SEMX_ERR_SHAPE
    assert status("semx_layer_norm_fwd", eps=-1.0) == _lib.SEMX_ERR_SHAPE
    assert status("semx_layer_norm_fwd", x=256, y=256, residual=256) == _lib.SEMX_ERR_NULL
    assert status("semx_layer_norm_fwd", x=258, y=256) == _lib.SEMX_ERR_ALIGN
    assert status("semx_layer_norm_fwd", x=257, y=256, x_bf16=1) == _lib.SEMX_ERR_ALIGN
    assert status("semx_layer_norm_bwd", sum=256) == _lib.SEMX_ERR_NULL
    assert status("semx_layer_norm_bwd", sum=256, mean=256, rstd=256, dy=256, dx=256, dweight=256) == _lib.SEMX_ERR_WORKSPACE


@pytest.mark.gpu
def test_argument_checks_on_cuda_tensors():
    from semambaxlinoss_b200.layer_norm import layer_norm

    x = torch.randn(2, 8, device=cuda())
    for bad in (dict(x=x.half()), dict(x=x, weight=x[0, :4]), dict(x=x, bias=x[0, :4]), dict(x=x, weight=x[0].cpu()),
                dict(x=x, residual=x[:1]), dict(x=x, residual=x.half()), dict(x=x[:, :0]), dict(x=x, out_dtype=torch.float16)):
        with pytest.raises(ValueError):
            layer_norm(bad["x"], bad.get("weight"), bad.get("bias"), residual=bad.get("residual"),
                       out_dtype=bad.get("out_dtype"))
    with pytest.raises(RuntimeError):
        layer_norm(torch.randn(1, 32769, device=x.device), None)
