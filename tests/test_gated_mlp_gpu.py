"""Gated projection on the GPU against the float64 oracle: rows from one to several tiles, odd and
narrow widths, strides, both types and activations, every combination of wanted gradients, streams
and captured graphs, the module, and the block that runs it behind the gated recurrence.

Tolerances, in units of eps = 2^-24 times the same sums over absolute values (the oracle's sizes). An
addition inside the tensor cores may cut instead of round: 2 eps. One product of depth K is K additions
in bf16 and 6 K in fp32, whose parts leave out 3 products of at most 2^-26 each (1 eps in all):
n(K) = 2 K (12 K) + 1.

* h: n(D) on u and g, activation and products 24 eps: n(D) + 24.
* dx: du and dg are n(D) + 32 off and, in bf16, rounded once more (2^-8 of their own size); the second
  product adds n(2 H). dw: n(rows) instead. db: a sum of `rows` terms.
* a result stored in bf16: half a step more, 2^-8 relative.
"""
from __future__ import annotations

import pytest
import torch

from oracle import gated_mlp as ogm
from tests.parity import cuda, gen, randn

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24
HALF = {torch.float32: EPS, torch.bfloat16: 2.0 ** -8}
SHAPES = [(1, 8, 1), (2, 64, 32), (3, 100, 7), (8, 2100, 33), (9, 64, 32), (33, 40, 24), (130, 72, 136), (129, 65, 33),
          (300, 257, 130), (1000, 64, 256), (257, 520, 264), (64, 2048, 40), (5000, 32, 16), (128, 64, 64),
          (1, 4096, 300), (5, 2056, 1030), (16, 136, 77), (17, 1000, 90)]


def _n(K, dtype):
    return (2 if dtype == torch.bfloat16 else 12) * K + 1


def _near(got, want, tol, dtype, what):
    got = got.detach().double().cpu().reshape(want.shape)
    tol = tol + HALF[dtype] * want.abs() + 2.0 ** -126
    over = (got - want).abs() - tol
    assert bool((over <= 0).all()), f"{what}: over by {over.max().item():.3e} at {int(over.argmax())}, " \
        f"max error {(got - want).abs().max().item():.3e} of {want.abs().max().item():.3e}"


def _operands(rows, D, H, dtype, seed, bias=True):
    g = gen(seed)
    x, w = randn((rows, D), g).to(dtype), randn((2 * H, D), g, scale=D ** -0.5).to(dtype)
    return x, w, randn((2 * H,), g, scale=0.3).to(dtype) if bias else None, randn((rows, H), g).to(dtype)


def _check(got, want, rows, D, H, dtype):
    part = HALF[dtype] if dtype == torch.bfloat16 else EPS  # of du and dg as the products read them
    for name, v in got.items():
        if name == "h":
            value, size = want["h"]
            _near(v, value, (_n(D, dtype) + 24) * EPS * size, dtype, name)
            continue
        value, size, plain = want[name]
        tol = (_n(D, dtype) + 32) * EPS * size
        if name == "db":
            tol = tol + rows * EPS * plain
        else:
            tol = tol + (part + _n(2 * H if name == "dx" else rows, dtype) * EPS) * plain
        _near(v, value, tol, dtype, name)


@pytest.mark.parametrize("rows,D,H", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("act,bias", [("silu", False), ("gelu", True)])
def test_forward(rows, D, H, dtype, act, bias):
    from semambaxlinoss_b200.gated_mlp import gated_linear

    x, w, b, _ = _operands(rows, D, H, dtype, rows + D, bias)
    h = gated_linear(x.to(cuda()), w.to(cuda()), None if b is None else b.to(cuda()), activation=act)
    want = ogm.gated(x.double(), w.double(), None if b is None else b.double(), act)
    assert h.shape == (rows, H) and h.dtype == dtype
    _check({"h": h}, want, rows, D, H, dtype)


@pytest.mark.parametrize("rows,D,H", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("act,bias", [("silu", True), ("gelu", False)])
def test_training(rows, D, H, dtype, act, bias):
    from semambaxlinoss_b200.gated_mlp import gated_linear

    x, w, b, dh = _operands(rows, D, H, dtype, rows + H, bias)
    ins = [t.to(cuda()).requires_grad_() for t in (x, w, b) if t is not None]
    h = gated_linear(ins[0], ins[1], ins[2] if bias else None, activation=act)
    grads = torch.autograd.grad(h, ins, dh.to(cuda()))
    want = ogm.gated(x.double(), w.double(), b.double() if bias else None, act, dh.double())
    assert all(g.dtype == dtype and g.shape == t.shape for g, t in zip(grads, ins))
    _check(dict(zip(("h", "dx", "dw", "db"), (h,) + grads)), want, rows, D, H, dtype)


# Sizes whose oracle runs on the GPU, in 64 bits: tiles of every width, and a last round of tiles that runs in
# slices of the depth behind whole rounds, in each of the products.
@pytest.mark.parametrize("rows,D,H", [(600, 2112, 3300), (192, 512, 9472), (2600, 1700, 2000), (3000, 260, 2500),
                                      (4099, 640, 1000)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_many_tiles(rows, D, H, dtype):
    from semambaxlinoss_b200.gated_mlp import gated_linear

    x, w, b, dh = (t.to(cuda()) for t in _operands(rows, D, H, dtype, rows + D))
    ins = [t.requires_grad_() for t in (x, w, b)]
    h = gated_linear(*ins)
    grads = torch.autograd.grad(h, ins, dh)
    want = ogm.gated(x.detach().double(), w.detach().double(), b.detach().double(), "silu", dh.double())
    want = {k: tuple(t.cpu() for t in v) for k, v in want.items()}
    _check(dict(zip(("h", "dx", "dw", "db"), (h,) + grads)), want, rows, D, H, dtype)
    with torch.no_grad():
        assert torch.equal(gated_linear(x, w, b), h)


@pytest.mark.parametrize("wants", [(0,), (1,), (2,), (0, 2), (1, 2), (0, 1)])
def test_some_gradients(wants):
    """Each gradient alone is what it is beside the others."""
    from semambaxlinoss_b200.gated_mlp import gated_linear

    x, w, b, dh = (t.to(cuda()) for t in _operands(300, 72, 40, torch.bfloat16, 3))
    every = [t.clone().requires_grad_() for t in (x, w, b)]
    all_grads = torch.autograd.grad(gated_linear(*every), every, dh)
    some = [t.clone().requires_grad_(k in wants) for k, t in enumerate((x, w, b))]
    grads = torch.autograd.grad(gated_linear(*some), [some[k] for k in wants], dh)
    for k, g in zip(wants, grads):
        assert torch.equal(g, all_grads[k])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_and_shapes(dtype):
    """Rows of wider tensors at any offset, transposed and misaligned weights, leading dimensions."""
    from semambaxlinoss_b200.gated_mlp import gated_linear

    x, w, b, dh = _operands(60, 64, 24, dtype, 9)
    want = gated_linear(x.to(cuda()), w.to(cuda()), b.to(cuda()))
    wide = torch.full((60, 160), float("nan"), dtype=dtype, device=cuda())
    for off in (0, 8, 3):
        wide.fill_(float("nan"))
        wide[:, off:off + 64] = x.to(cuda())
        assert torch.equal(gated_linear(wide[:, off:off + 64], w.to(cuda()), b.to(cuda())), want), off
    turned = w.t().contiguous().to(cuda()).t()
    assert torch.equal(gated_linear(x.to(cuda()), turned, b.to(cuda())), want)
    flat = torch.zeros(w.numel() + 1, dtype=dtype, device=cuda())
    flat[1:] = w.to(cuda()).reshape(-1)
    assert torch.equal(gated_linear(x.to(cuda()), flat[1:].view(w.shape), b.to(cuda())), want)
    many = x.to(cuda()).view(5, 3, 4, 64)
    assert torch.equal(gated_linear(many, w.to(cuda()), b.to(cuda())), want.view(5, 3, 4, 24))
    turned = many.transpose(0, 2)  # rows at no single stride
    assert torch.equal(gated_linear(turned, w.to(cuda()), b.to(cuda())), want.view(5, 3, 4, 24).transpose(0, 2))
    one = x[:1].to(cuda())
    got = gated_linear(one.expand(60, 64), w.to(cuda()), b.to(cuda()))
    assert torch.equal(got, got[:1].expand(60, 24))
    xe, we = one.clone().requires_grad_(), w.to(cuda()).requires_grad_()
    dx, dw = torch.autograd.grad(gated_linear(xe.expand(60, 64), we), (xe, we), dh.to(cuda()))
    assert dx.shape == (1, 64) and dw.shape == w.shape
    single = gated_linear(x[0].to(cuda()), w.to(cuda()), b.to(cuda()))
    assert single.shape == (24,)


@pytest.mark.parametrize("rows", [1, 2, 5, 8, 9, 12, 16, 17])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_few_strided_rows(rows, dtype):
    """Few rows of a wider tensor at any offset: the bits of the same rows alone, at two widths of D."""
    from semambaxlinoss_b200.gated_mlp import gated_linear

    for D, H in ((200, 19), (2308, 36)):
        x, w, b, _ = (t.to(cuda()) for t in _operands(rows, D, H, dtype, rows + D))
        for off, ld in ((0, D + 8), (4, D + 4), (3, D + 5)):
            wide = torch.full((rows, ld + off), float("nan"), dtype=dtype, device=cuda())
            wide[:, off:off + D] = x
            h = gated_linear(wide[:, off:off + D], w, b)
            want = ogm.gated(x.double().cpu(), w.double().cpu(), b.double().cpu(), "silu")
            _check({"h": h}, want, rows, D, H, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_saved_tensors_moved(dtype):
    """Operands whose rows are strided, kept elsewhere between the passes: they come back dense."""
    from semambaxlinoss_b200.gated_mlp import gated_linear

    x, w, b, dh = (t.to(cuda()) for t in _operands(150, 64, 24, dtype, 37))
    for off in (0, 3):
        wide = torch.full((150, 160), float("nan"), dtype=dtype, device=cuda())
        wide[:, off:off + 64] = x
        ins = [wide[:, off:off + 64].requires_grad_(), w.clone().requires_grad_(), b.clone().requires_grad_()]
        want = torch.autograd.grad(gated_linear(*ins), ins, dh)
        with torch.autograd.graph.save_on_cpu():
            h = gated_linear(*ins)
        got = torch.autograd.grad(h, ins, dh)
        assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_empty():
    from semambaxlinoss_b200.gated_mlp import gated_linear

    x = torch.zeros(0, 16, device=cuda(), requires_grad=True)
    w = torch.ones(8, 16, device=cuda(), requires_grad=True)
    b = torch.ones(8, device=cuda(), requires_grad=True)
    h = gated_linear(x, w, b)
    dx, dw, db = torch.autograd.grad(h.sum(), (x, w, b))
    assert h.shape == (0, 4) and dx.shape == x.shape and not dw.any() and not db.any()
    assert gated_linear(torch.zeros(2, 0, 16, device=cuda()), w.detach()).shape == (2, 0, 4)


def test_numbers_that_are_none():
    """NaN and infinities of one row or weight stay in what depends on them."""
    from semambaxlinoss_b200.gated_mlp import gated_linear

    for dtype in (torch.bfloat16, torch.float32):
        x, w, _, _ = _operands(140, 100, 36, dtype, 12, False)
        clean = gated_linear(x.to(cuda()), w.to(cuda()))
        x2 = x.clone()
        x2[3, 5], x2[130, 99] = float("nan"), float("inf")
        h = gated_linear(x2.to(cuda()), w.to(cuda()))
        keep = [r for r in range(140) if r not in (3, 130)]
        assert torch.equal(h[keep], clean[keep]) and torch.isnan(h[3]).all() and not torch.isfinite(h[130]).any()
        w2 = w.clone()
        w2[35] = float("nan")  # the value's last row, in front of the gate's first
        h = gated_linear(x.to(cuda()), w2.to(cuda()))
        assert torch.equal(h[:, :35], clean[:, :35]) and torch.isnan(h[:, 35]).all()
        big = gated_linear(torch.full((20, 8), 3.3e38).to(dtype).to(cuda()), torch.full((4, 8), 1e-38).to(dtype).to(cuda()))
        assert torch.isfinite(big).all()


def test_gradients_against_differences():
    from semambaxlinoss_b200.gated_mlp import gated_linear

    x, w, b, dh = (t.double() for t in _operands(70, 48, 20, torch.float32, 17))
    for act in ("silu", "gelu"):
        dev = [t.float().to(cuda()).requires_grad_() for t in (x, w, b)]
        grads = torch.autograd.grad(gated_linear(*dev, activation=act), dev, dh.float().to(cuda()))
        g = gen(5)
        for k in range(3):
            v = randn(tuple((x, w, b)[k].shape), g)
            up, down = [x, w, b], [x, w, b]
            up[k], down[k] = up[k] + 1e-5 * v, down[k] - 1e-5 * v
            diff = ((ogm.gated(*up, act)["h"][0] - ogm.gated(*down, act)["h"][0]) * dh).sum() / 2e-5
            got = (grads[k].double().cpu() * v).sum()
            assert abs(got - diff) <= 1e-4 * (grads[k].double().cpu() * v).abs().sum(), (act, k)


def test_repeats_streams_and_graphs():
    """The same bits from run to run, on two streams at once, and from replayed graphs of forward and
    training passes that share memory."""
    from semambaxlinoss_b200.gated_mlp import gated_linear

    for rows, D, H, dtype in ((200, 520, 136, torch.bfloat16), (700, 65, 33, torch.float32)):
        x, w, b, dh = (t.to(cuda()) for t in _operands(rows, D, H, dtype, 21))

        def train():
            v = [t.detach().requires_grad_() for t in (x, w, b)]
            h = gated_linear(*v)
            return (h,) + torch.autograd.grad(h, v, dh)

        want = [t.detach().clone() for t in train()]
        for _ in range(3):
            assert all(torch.equal(p, q) for p, q in zip(train(), want))
        torch.cuda.synchronize()
        got = []
        for _ in range(2):
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                got.append(train())
        torch.cuda.synchronize()
        for res in got:
            assert all(torch.equal(p, q) for p, q in zip(res, want))
        pool, graphs = torch.cuda.graph_pool_handle(), []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, pool=pool):
                res = train()
            graphs.append((graph, res))
        for graph, res in graphs:
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(res, want))


def test_autocast():
    """fp32 parameters under bf16 autocast: the results of cast ones, gradients in fp32."""
    from semambaxlinoss_b200.gated_mlp import gated_linear

    x, w, b, dh = (t.to(cuda()) for t in _operands(100, 64, 24, torch.float32, 31))
    ins = [t.requires_grad_() for t in (x, w, b)]
    with torch.autocast("cuda", dtype=torch.bfloat16):
        h = gated_linear(*ins)
    assert h.dtype == torch.bfloat16
    grads = torch.autograd.grad(h, ins, dh.to(torch.bfloat16))
    cast = [x.detach().to(torch.bfloat16).requires_grad_(), w.detach().to(torch.bfloat16).requires_grad_(),
            b.detach().requires_grad_()]
    plain = gated_linear(*cast)
    want = torch.autograd.grad(plain, cast, dh.to(torch.bfloat16))
    assert torch.equal(h, plain)
    for g, q in zip(grads, want):
        assert g.dtype == torch.float32 and torch.equal(g, q.float())


def test_refusals():
    from semambaxlinoss_b200.gated_mlp import gated_linear

    x, w, b = torch.zeros(4, 16, device=cuda()), torch.zeros(12, 16, device=cuda()), torch.zeros(12, device=cuda())
    for bad, what in ((dict(weight=w[:11]), "weight"), (dict(weight=w[:, :15]), "weight"), (dict(weight=w[0]), "weight"),
                      (dict(weight=w.to(torch.bfloat16)), "weight"), (dict(weight=w.cpu()), "weight"),
                      (dict(bias=b[:6]), "bias"), (dict(bias=b.double()), "bias"), (dict(bias=b.cpu()), "bias"),
                      (dict(activation="relu"), "activation"), (dict(x=x.double()), "dtype"), (dict(x=x.half()), "dtype"),
                      (dict(x=x[:, :0], weight=w[:, :0]), "features")):
        with pytest.raises(ValueError, match=what):
            gated_linear(**dict(dict(x=x, weight=w, bias=b), **bad))
    with torch.autocast("cuda", dtype=torch.float16), pytest.raises(ValueError, match="dtype"):
        gated_linear(x, w, b)
    import torch.autograd.forward_ad as fwad

    with fwad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        gated_linear(fwad.make_dual(x, torch.ones_like(x)), w, b)
    xr = x.clone().requires_grad_()
    (g,) = torch.autograd.grad(gated_linear(xr, w, b).sum(), xr, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), xr)


def test_no_wait_gave_up():
    from semambaxlinoss_b200 import _lib

    assert _lib.tc_timeouts() == 0


def _block(cfg, dim, dtype=torch.float32, seed=0):
    from semambaxlinoss_b200.mamba_block import create_block

    torch.manual_seed(seed)
    return create_block(dim, dict({"d_state": 4, "d_conv": 4, "expand": 2}, **cfg)).to(cuda(), dtype)


@pytest.mark.parametrize("dim,mlp", [(64, {}), (33, {"hidden_features": 50, "activation": "gelu", "bias": True})])
def test_module_matches_its_formula(dim, mlp):
    from semambaxlinoss_b200.gated_mlp import GatedMLP

    torch.manual_seed(1)
    m = GatedMLP(dim, **mlp).to(cuda())
    assert m.hidden_features == mlp.get("hidden_features", 256)
    x = randn((3, 50, dim), gen(2)).float().to(cuda())
    want = ogm.gated(x.double().cpu().view(-1, dim), m.fc1.weight.detach().double().cpu(),
                     None if m.fc1.bias is None else m.fc1.bias.detach().double().cpu(), m.activation)["h"][0]
    want = torch.nn.functional.linear(want, m.fc2.weight.detach().double().cpu(),
                                      None if m.fc2.bias is None else m.fc2.bias.detach().double().cpu())
    got = m(x)
    assert got.shape == x.shape
    assert (got.detach().double().cpu().view(-1, dim) - want).abs().max() <= 1e-5 * want.abs().max()


def test_block_trains_prompts_and_steps():
    """A block of the gated recurrence and the feed-forward half: a training pass with every gradient;
    a packed prompt with a cache, then single tokens, as the whole sequences."""
    dim = 40
    m = _block({"ssm": "gated_lru", "mlp": {}}, dim, seed=4)
    g = gen(41)
    x = randn((2, 150, dim), g).float().to(cuda()).requires_grad_()
    h, res = m(x)
    ((h + res) * randn((2, 150, dim), g).float().to(cuda())).sum().backward()
    assert x.grad.any() and torch.isfinite(x.grad).all()
    for name, p in m.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all() and p.grad.any(), name
    with torch.no_grad():
        whole = [sum(m(x[k:k + 1])) for k in range(2)]
        cache = m.mixer.allocate_cache(3)
        slots = torch.tensor([2, 0], dtype=torch.int32, device=cuda())
        fresh = torch.ones(2, dtype=torch.bool, device=cuda())
        cu = torch.tensor([0, 148, 268], dtype=torch.int32, device=cuda())
        packed = torch.cat([x[0, :148], x[1, :120]])
        y = sum(m(packed, cu_seqlens=cu, cache=cache, slots=slots, fresh=fresh))
        assert torch.allclose(y[:148], whole[0][0, :148], rtol=1e-4, atol=1e-4)
        assert torch.allclose(y[148:], whole[1][0, :120], rtol=1e-4, atol=1e-4)
        for t in range(2):
            tok = torch.stack([x[0, 148 + t], x[1, 120 + t]])[:, None]
            y = sum(m(tok, cache=cache, slots=slots))
            assert torch.allclose(y[0, 0], whole[0][0, 148 + t], rtol=1e-4, atol=1e-4)
            assert torch.allclose(y[1, 0], whole[1][0, 120 + t], rtol=1e-4, atol=1e-4)


def test_decoding_graph_of_the_block():
    """Single tokens of the block in a replayed graph: what the eager calls give."""
    dim = 48
    m = _block({"ssm": "gated_lru", "mlp": {"hidden_features": 128}}, dim, torch.bfloat16, seed=6)
    m.mixer.rate.data = m.mixer.rate.data.float()
    toks = randn((6, 3, 1, dim), gen(7)).to(torch.bfloat16).to(cuda())
    with torch.no_grad():
        cache = m.mixer.allocate_cache(3)
        want = [sum(m(t, cache=cache)) for t in toks]
        cache = m.mixer.allocate_cache(3)
        static = toks[0].clone()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            sum(m(static, cache=cache))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = sum(m(static, cache=cache))
        cache.window.zero_()
        cache.state.zero_()
        for t, w in zip(toks, want):
            static.copy_(t)
            graph.replay()
            assert torch.equal(out, w)


@pytest.mark.parametrize("bidirectional", [True, False])
def test_mamba_block_with_feed_forward(bidirectional):
    from semambaxlinoss_b200.mamba_block import MambaBlock

    torch.manual_seed(8)
    cfg = {"ssm": "gated_lru", "d_state": 4, "d_conv": 3, "expand": 2, "mlp": {}, "bidirectional": bidirectional}
    m = MambaBlock(32, cfg).to(cuda())
    x = randn((2, 80, 32), gen(9)).float().to(cuda()).requires_grad_()
    y = m(x)
    assert y.shape == (2, 80, 64 if bidirectional else 32)
    y.sum().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in m.parameters())
