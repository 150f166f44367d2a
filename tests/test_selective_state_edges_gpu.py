"""Selective state operators on the GPU at the ends of what a call may ask for, against the
float64 oracle. Tolerances as derived in test_selective_state_gpu.py."""
from __future__ import annotations

import pytest
import torch

import tests.test_selective_state_gpu as base
from oracle import selective_state as oss
from tests.parity import cuda, gen, randn
from tests.test_selective_state_gpu import _batched, _near, _scan_problem, _seqs, _strided

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["short", "ragged", "long"])
@pytest.mark.parametrize("ch,N,G,pad", [(64, 16, 1, 0), (65, 16, 1, 3), (200, 4, 2, 0), (12, 128, 2, 0)])
@pytest.mark.parametrize("dtt", [torch.bfloat16, torch.float32])
def test_gate_gradient_is_rounded_once(kind, ch, N, G, pad, dtt):
    """bf16 rows: dz = dy v silu'(z) from a v in fp32, so dz has the forward's and the adjoint's
    fp32 error, (16 len + 128) 2^-24 of its terms, and the one rounding that stores it."""
    from semambaxlinoss_b200.selective_state import selective_state_scan

    cu, rows = _seqs(kind)
    g = gen(ch + N)
    t = _scan_problem(rows, ch, N, G, g, torch.bfloat16, dtt)
    dy = randn((rows, ch), g).bfloat16()
    v = {k: _batched(kind, _strided(u, pad))[0] if k in ("x", "dt", "B", "C", "z") else u.to(cuda()) for k, u in t.items()}
    z = v["z"].requires_grad_()
    y = selective_state_scan(v["x"], v["dt"], v["A"], v["B"], v["C"], v["D"], z, v["dt_bias"],
                             cu_seqlens=_batched(kind, t["x"])[1])
    (dz,) = torch.autograd.grad(y, z, _batched(kind, dy.to(cuda()))[0])
    d = {k: u.double() for k, u in t.items()}
    args = (d["x"], d["dt"], d["A"], d["B"], d["C"], cu, d["D"], d["z"], d["dt_bias"])
    out, size = oss.scan(*args, dy=dy.double()), oss.scan(*args, dy=dy.double(), absolute=True)
    longest = max(b - a for a, b in zip(cu[:-1], cu[1:]))
    _near(dz, out["dz"], size["dz"], 16 * longest + 128, torch.bfloat16, "dz")


@pytest.fixture
def poisoned():
    """Every fresh allocation starts as NaN, so that what a kernel leaves unwritten shows."""
    before = torch.are_deterministic_algorithms_enabled(), torch.utils.deterministic.fill_uninitialized_memory
    torch.use_deterministic_algorithms(True, warn_only=True)
    torch.utils.deterministic.fill_uninitialized_memory = True
    yield
    torch.use_deterministic_algorithms(before[0])
    torch.utils.deterministic.fill_uninitialized_memory = before[1]


# Offsets that begin above 0: short sequences, more unused rows than pieces, sequences that are cut
# into pieces, a batch of which one sequence is cut (it fills the GPU), none at all.
FRONT = {"short": ([5, 12, 20], 24), "far": ([700, 701, 703, 703, 720], 900), "pieces": ([37, 437, 440], 443),
         "outlier": ([3, 303] + [303 + 3 * i for i in range(1, 310)], 1235), "none": ([4, 4], 9), "end": ([9, 9, 9], 9)}


@pytest.mark.parametrize("kind", FRONT)
@pytest.mark.parametrize("ch,N,G", [(40, 16, 1), (33, 5, 3), (8, 128, 2)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_in_front_of_the_first_sequence(kind, ch, N, G, dtype, poisoned):
    """A slice of a larger batch: rows that no sequence owns, in front and behind, come out as
    zeros in outputs and gradients, and reach nothing else."""
    from semambaxlinoss_b200.selective_state import selective_state_scan, short_conv

    cu, rows = FRONT[kind]
    S, g = len(cu) - 1, gen(ch + N)
    t = _scan_problem(rows, ch, N, G, g, dtype)
    w, b, dy = randn((ch, 4), g, scale=0.5).float(), randn((ch,), g).float(), randn((rows, ch), g).to(dtype)
    cud = torch.tensor(cu, dtype=torch.int32, device=cuda())
    unused = torch.tensor([i < cu[0] or i >= cu[-1] for i in range(rows)])
    t["x"][unused], dy[unused] = float("nan"), float("nan")
    v = {k: u.to(cuda()).requires_grad_() for k, u in dict(t, w=w, b=b).items()}
    clean = {k: torch.where(unused.view((-1,) + (1,) * (u.dim() - 1)), torch.zeros_like(u), u) if u.shape[0] == rows and k not in ("A", "D", "dt_bias")
             else u for k, u in t.items()}
    d = {k: u.double() for k, u in clean.items()}
    dy64 = torch.where(unused[:, None], torch.zeros_like(dy), dy).double()

    y = short_conv(v["x"], v["w"], v["b"], cu_seqlens=cud)
    got = dict(zip(("dx", "dw", "db"), torch.autograd.grad(y, (v["x"], v["w"], v["b"]), dy.to(cuda()))), y=y)
    out = oss.conv(d["x"], w.double(), b.double(), cu, dy=dy64)
    size = oss.conv(d["x"].abs(), w.double().abs(), b.double().abs(), cu, False, dy=dy64.abs())
    grow = 1.1 + size["y"].amax()
    _near(got["y"], out["y"], size["y"], 64, dtype, "conv y")
    _near(got["dx"], out["dx"], size["dx"] * grow, 64, dtype, "conv dx")
    _near(got["dw"], out["dw"], size["aw"] * grow, 64 + min(rows, 64) + 64, torch.float32, "conv dw")
    _near(got["db"], out["db"], size["ab"] * grow, 64 + min(rows, 64) + 64, torch.float32, "conv db")
    for k in ("y", "dx"):
        assert not got[k].cpu()[unused].any(), k  # NaN counts as true

    names = ("x", "dt", "A", "B", "C", "D", "z", "dt_bias")
    y = selective_state_scan(*[v[k] for k in names[:5]], D=v["D"], z=v["z"], dt_bias=v["dt_bias"], cu_seqlens=cud)
    got = dict(zip(names, torch.autograd.grad(y, [v[k] for k in names], dy.to(cuda()))))
    args = (d["x"], d["dt"], d["A"], d["B"], d["C"], cu, d["D"], d["z"], d["dt_bias"])
    out, size = oss.scan(*args, dy=dy64), oss.scan(*args, dy=dy64, absolute=True)
    longest = max(q - p for p, q in zip(cu[:-1], cu[1:]))
    _near(y, out["y"], size["y"], 8 * longest + 64, dtype, "y")
    assert not y.cpu()[unused].any()
    for k in names:
        n = 16 * longest + 128 + (ch if k in ("B", "C") else rows if k in ("A", "D", "dt_bias") else 0)
        _near(got[k], out["d" + k], size["d" + k], n, got[k].dtype, "d" + k)
        assert k in ("A", "D", "dt_bias") or not got[k].cpu()[unused].any(), k

    with torch.no_grad():
        for call, shape, dt in ((lambda p: short_conv(v["x"], v["w"], v["b"], cu_seqlens=cud, state=p), (3, ch), dtype),
                                (lambda p: selective_state_scan(*[v[k] for k in names[:5]], D=v["D"], z=v["z"],
                                                                dt_bias=v["dt_bias"], cu_seqlens=cud, state=p), (ch, N),
                                 torch.float32)):
            y = call(torch.zeros((S,) + shape, dtype=dt, device=cuda())).cpu()
            assert not y[unused].any() and bool(torch.isfinite(y).all())


def test_forward_mode_tangents_are_refused():
    """Every operand of every operator: a tangent is refused, not lost, and no state moves."""
    from torch.autograd import forward_ad

    from semambaxlinoss_b200.layer_norm import LayerNorm, layer_norm
    from semambaxlinoss_b200.selective_state import (selective_state_scan, selective_state_step, short_conv,
                                                     short_conv_step)

    dev, ch, N = cuda(), 8, 4
    r = lambda *s: torch.randn(*s, device=dev)  # noqa: E731
    x, BC, vec = r(2, 5, ch), r(2, 5, N), r(ch)
    conv = dict(x=x, weight=r(ch, 4), bias=vec)
    scan = dict(x=x, dt=x.clone(), A=-r(ch, N).abs(), B=BC, C=BC.clone(), D=vec, z=x.clone(), dt_bias=vec.clone())
    one = {k: u[:, 0] if k in ("x", "dt", "B", "C", "z") else u for k, u in scan.items()}
    window, state = torch.zeros(2, 3, ch, device=dev), torch.zeros(2, ch, N, device=dev)
    calls = [(short_conv, conv), (short_conv, dict(conv, state=window)), (selective_state_scan, scan),
             (selective_state_scan, dict(scan, state=state)), (selective_state_step, dict(one, state=state)),
             (short_conv_step, dict(conv, x=x[:, 0], state=window)),
             (layer_norm, dict(x=x, weight=vec, bias=vec.clone(), residual=x.clone())),
             (LayerNorm(ch, device=dev), dict(x=x, residual=x.clone()))]
    for call, kw in calls:
        with torch.no_grad():
            call(**kw)
        window.zero_(), state.zero_()
        for name in kw:
            with forward_ad.dual_level(), torch.no_grad(), pytest.raises(NotImplementedError):
                call(**dict(kw, **{name: forward_ad.make_dual(kw[name], torch.ones_like(kw[name]))}))
            assert not window.any() and not state.any(), (call, name)


# Rows, groups and modes on four elements, so that every operand is read four at a time, with 8, 16
# and 32 lanes per channel (a lane holds four modes), full and partly used, and the gate.
VECTORS = [(264, 32, 1, 4), (48, 28, 2, 0), (16, 64, 1, 0), (40, 36, 1, 8), (24, 128, 2, 8), (32, 100, 1, 0)]


@pytest.mark.parametrize("kind", ["one", "short", "even", "ragged", "long"])
@pytest.mark.parametrize("ch,N,G,pad", VECTORS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_vector_rows_of_many_modes_training(kind, ch, N, G, pad, dtype):
    base.test_scan_training(kind, ch, N, G, pad, True, True, True, dtype, None)


@pytest.mark.parametrize("kind", ["one", "short", "even", "ragged", "long", "many"])
@pytest.mark.parametrize("ch,N,G", [v[:3] for v in VECTORS])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_vector_rows_of_many_modes_prompts(kind, ch, N, G, dtype):
    base.test_scan_prompts(kind, ch, N, G, dtype)


@pytest.mark.parametrize("S", [1, 9, 150])
@pytest.mark.parametrize("ch,N,G", [v[:3] for v in VECTORS])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_vector_rows_of_many_modes_tokens(S, ch, N, G, dtype):
    base.test_single_tokens(S, ch, N, G, 4, dtype)


DIFF = ("x", "w", "b", "dt", "A", "B", "C", "D", "z", "dt_bias")


def _difference_problem():
    g, rows, ch, N = gen(11), 24, 40, 16
    t = _scan_problem(rows, ch, N, 2, g, torch.float32)
    t |= {"w": randn((ch, 4), g).float(), "b": randn((ch,), g).float()}
    return t, randn((rows, ch), g).float(), [0, 7, 7, 20]


def _allowed(slope, y, weight, h):
    """Difference against slope: (8 len + 64) 2^-24 of the outputs' terms, 4 for sums that cancel, over the
    step; and the third derivative. A direction of size 0.3 in every step and rate moves the
    logarithm of 13 poles' product by at most 13 x 0.3 = 4, so it is at most 4^3 / 6 of the slope's terms
    in h^2; the products with the other operands double it a few times: 64."""
    return (8 * 13 + 64) * 2.0 ** -24 / h * 4 * (y.abs() * weight.abs()).sum() + 64 * h * h * slope


@pytest.mark.parametrize("name", DIFF)
def test_each_gradient_against_differences(name):
    """The operators' own outputs moved along the sign of one operand's gradient, where the slope is the sum
    of its absolute values: without the gradient, or with a quarter of it wrong, the test fails."""
    from semambaxlinoss_b200.selective_state import selective_state_scan, short_conv

    t, weight, cu = _difference_problem()
    t, weight, cud = {k: u.to(cuda()) for k, u in t.items()}, weight.to(cuda()), torch.tensor(cu, dtype=torch.int32, device=cuda())

    def value(v):
        u = short_conv(v["x"], v["w"], v["b"], cu_seqlens=cud)
        return selective_state_scan(u, v["dt"], v["A"], v["B"], v["C"], v["D"], v["z"], v["dt_bias"], cu_seqlens=cud)

    leaf = t[name].clone().requires_grad_()
    (grad,) = torch.autograd.grad(value(dict(t, **{name: leaf})), leaf, weight)
    move, h = 0.3 * grad.sign(), 2.0 ** -7
    slope = (grad.double() * move.double()).sum()
    up, down = (value(dict(t, **{name: t[name] + s * h * move})).double() for s in (1, -1))
    tol = _allowed(slope, up, weight, h)
    assert tol < 0.25 * slope
    assert (((up - down) * weight).sum() / (2 * h) - slope).abs() <= tol


def test_pieces_hold_the_precision_of_one_pass():
    """One sequence of 500 rows, cut into pieces both ways, against 64 bits in the 2-norm. Steps of 0.13
    and rates of 1 keep a state for about 10 steps: 10 roundings of the state, 4 eps of each pole,
    the same again in the adjoint, in the 2-norm below 32 eps; a piece that starts from a wrong
    state is off by hundredths."""
    from semambaxlinoss_b200.selective_state import selective_state_scan

    g, L, ch, N = gen(29), 500, 96, 16
    t = _scan_problem(L, ch, N, 1, g, torch.float32)
    dy = randn((L, ch), g).float()
    names = ("x", "dt", "A", "B", "C", "D", "z", "dt_bias")
    v = {k: (u[None] if k in ("x", "dt", "B", "C", "z") else u).to(cuda()).requires_grad_() for k, u in t.items()}
    y = selective_state_scan(*[v[k] for k in names[:5]], D=v["D"], z=v["z"], dt_bias=v["dt_bias"])
    grads = torch.autograd.grad(y, [v[k] for k in names], dy[None].to(cuda()))
    d = {k: u.double() for k, u in t.items()}
    out = oss.scan(d["x"], d["dt"], d["A"], d["B"], d["C"], [0, L], d["D"], d["z"], d["dt_bias"], dy=dy.double())
    for name, got in zip(("y",) + tuple("d" + k for k in names), (y,) + grads):
        want = out[name]
        off = (got.detach().double().cpu().reshape(want.shape) - want).norm() / want.norm()
        assert off <= 32 * 2.0 ** -24, (name, off)


@pytest.mark.parametrize("width,groups", [(64, 1), (128, 2)])
def test_block_with_vector_rows(width, groups):
    """The block as a whole where the projections' rows allow four elements at a time (dt_rank 4 and 8), with
    every gradient; 1e-4 of the largest value as for the other block tests."""
    from semambaxlinoss_b200.mamba_block import create_block

    torch.manual_seed(width)
    cfg = {"ssm": "selective_state", "d_state": 16, "d_conv": 4, "expand": 2, "ssm_params": {"n_groups": groups}}
    block = create_block(width, cfg, rms_norm=False, fused_add_norm=True)
    with torch.no_grad():
        for p in block.parameters():
            p.add_(torch.randn(p.shape) * 0.05)
    block, rank, GN = block.to(cuda()), width // 16, groups * 16
    g, cu = gen(width), [2, 19, 20, 60]
    x, r, dy, ds = (randn((61, width), g).float() for _ in range(4))
    p = {k: u.detach().double().cpu().requires_grad_() for k, u in block.named_parameters()}
    x64, r64 = x.double().requires_grad_(), r.double().requires_grad_()
    s64 = x64 + r64
    xz = torch.nn.functional.layer_norm(s64, (width,), p["norm.weight"], p["norm.bias"]) @ p["mixer.in_proj.weight"].t()
    u, z = xz.chunk(2, -1)
    u = oss.conv(u, p["mixer.conv1d.weight"][:, 0], p["mixer.conv1d.bias"], cu)["y"]
    rows = u @ p["mixer.x_proj.weight"].t()
    B, C = (rows[:, rank + i * GN:rank + (i + 1) * GN].unflatten(-1, (groups, 16)) for i in range(2))
    y64 = oss.scan(u, rows[:, :rank] @ p["mixer.dt_proj.weight"].t(), -torch.exp(p["mixer.A_log"]), B, C, cu, p["mixer.D"], z,
                   p["mixer.dt_proj.bias"])["y"] @ p["mixer.out_proj.weight"].t()
    want = torch.autograd.grad((y64 * dy).sum() + (s64 * ds).sum(), [x64, r64] + list(p.values()))
    xd, rd = x.to(cuda()).requires_grad_(), r.to(cuda()).requires_grad_()
    y, s = block(xd, rd, cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=cuda()))
    got = torch.autograd.grad((y, s), [xd, rd] + list(block.parameters()), (dy.to(cuda()), ds.to(cuda())))
    for name, a, b in zip(["y", "s", "x", "r"] + list(p), (y, s) + got, (y64, s64) + want):
        err = (a.detach().double().cpu() - b.detach()).abs().max() / b.detach().abs().max()
        assert err <= 1e-4, (name, err)


@pytest.mark.parametrize("ch,N,G", [(64, 16, 1), (33, 5, 3)])
def test_fp32_steps_beside_bf16_rows(ch, N, G):
    """Prompts and single tokens whose step projection stayed in fp32."""
    from semambaxlinoss_b200.selective_state import selective_state_scan, selective_state_step

    S, L, g = 5, 9, gen(ch)
    t = _scan_problem(S * L, ch, N, G, g, torch.bfloat16, torch.float32)
    start, cu = randn((S, ch, N), g).float(), [L * s for s in range(S + 1)]
    v = {k: (u.view((S, L) + u.shape[1:]) if k in ("x", "dt", "B", "C", "z") else u).to(cuda()) for k, u in t.items()}
    d = {k: u.double() for k, u in t.items()}
    state = start.to(cuda())
    y = selective_state_scan(*[v[k] for k in ("x", "dt", "A", "B", "C", "D", "z", "dt_bias")], state=state)
    args = (d["x"], d["dt"], d["A"], d["B"], d["C"], cu, d["D"], d["z"], d["dt_bias"])
    h0 = [u.double() for u in start]
    out, size = oss.scan(*args, h0=h0), oss.scan(*args, h0=h0, absolute=True)
    _near(y, out["y"], size["y"], 8 * L + 64, torch.bfloat16, "y")
    _near(state, torch.stack(out["h"]), torch.stack(size["h"]), 8 * L + 64, torch.float32, "state")
    one = {k: u[:, 0] if k in ("x", "dt", "B", "C", "z") else u for k, u in v.items()}  # rows at L times the stride
    state = start.to(cuda())
    y = selective_state_step(*[one[k] for k in ("x", "dt", "A", "B", "C")], state, one["D"], one["z"], one["dt_bias"])
    first = {k: u[::L] if k in ("x", "dt", "B", "C", "z") else u for k, u in d.items()}
    args = (first["x"], first["dt"], first["A"], first["B"], first["C"], list(range(S + 1)), first["D"], first["z"], first["dt_bias"])
    out, size = oss.scan(*args, h0=h0), oss.scan(*args, h0=h0, absolute=True)
    _near(y, out["y"], size["y"], 72, torch.bfloat16, "token")
    _near(state, torch.stack(out["h"]), torch.stack(size["h"]), 72, torch.float32, "token state")


def test_slots_named_again_far_behind():
    """Two sequences of one slot that different CTAs run: the first has it, the later ones are refused."""
    S, dev = 700, cuda()
    again = {350: 3, 699: 3, 698: 697, 17: 16}
    for name, call, shape in base._ops(S):
        pool = torch.randn((S,) + shape, device=dev)
        good = torch.arange(S, dtype=torch.int32, device=dev)
        bad = good.clone()
        for s, other in again.items():
            bad[s] = other
        p0, p1 = pool.clone(), pool.clone()
        want, got = call(p0, good), call(p1, bad)
        for s in range(S):
            p0[s] = pool[s] if s in again else p0[s]
        refused = torch.tensor([s in again for s in range(S)], device=dev)
        assert torch.isnan(got[refused]).all() and torch.equal(got[~refused], want[~refused]), name
        assert torch.equal(p0, p1), name


def test_no_steps_and_inference_mode():
    from semambaxlinoss_b200.selective_state import selective_state_scan, short_conv

    dev, ch, N = cuda(), 16, 4
    x, B = torch.empty(3, 0, ch, device=dev, requires_grad=True), torch.empty(3, 0, N, device=dev)
    A, w = (-torch.rand(ch, N, device=dev)).requires_grad_(), torch.rand(ch, 4, device=dev, requires_grad=True)
    y = selective_state_scan(short_conv(x, w), x, A, B, B, z=x)
    assert y.shape == x.shape
    dx, dA, dw = torch.autograd.grad(y, (x, A, w), torch.empty_like(y))
    assert dx.shape == x.shape and not dA.any() and not dw.any()
    state = torch.ones(3, ch, N, device=dev)
    with torch.no_grad():
        selective_state_scan(x, x, A, B, B, state=state, fresh=torch.tensor([True, False, True], device=dev))
    assert not state[[0, 2]].any() and bool((state[1] == 1).all())
    x, B = torch.randn(2, 9, ch, device=dev), torch.randn(2, 9, N, device=dev)
    with torch.no_grad():
        want = selective_state_scan(short_conv(x, w), x, A, B, B)
    with torch.inference_mode():
        assert torch.equal(selective_state_scan(short_conv(x, w), x, A, B, B), want)


def test_a_captured_prompt_takes_other_offsets():
    """A packed prompt captured once and replayed with other offsets, slots and fresh flags (a long sequence
    where short ones were, rows in front of the first): what plain calls give, bit for bit."""
    from semambaxlinoss_b200.selective_state import selective_state_scan, short_conv

    g, rows, S, ch, N, dev = gen(31), 700, 6, 72, 16, cuda()
    t = {k: u.to(dev) for k, u in _scan_problem(rows, ch, N, 1, g, torch.bfloat16).items()}
    w = torch.randn(ch, 4, device=dev)
    plans = [([0, 5, 9, 9, 30, 600, 690], [3, 0, 7, 1, 2, 5], [1, 0, 1, 0, 0, 1]),
             ([4, 650, 651, 652, 652, 652, 655], [7, 6, 5, 4, -1, 0], [0, 0, 0, 0, 1, 1]),
             ([0, 100, 200, 300, 400, 500, 700], [0, 1, 2, 2, 4, 9], [0] * 6)]
    cu, slots = (torch.zeros(n, dtype=torch.int32, device=dev) for n in (S + 1, S))
    fresh = torch.zeros(S, dtype=torch.bool, device=dev)
    window, state = torch.randn(8, 3, ch, device=dev).bfloat16(), torch.randn(8, ch, N, device=dev)

    def prompt(window, state):
        u = short_conv(t["x"], w, cu_seqlens=cu, state=window, slots=slots, fresh=fresh)
        return selective_state_scan(u, *[t[k] for k in ("dt", "A", "B", "C", "D", "z", "dt_bias")], cu_seqlens=cu,
                                    state=state, slots=slots, fresh=fresh)

    def plan(i):
        for buf, values in zip((cu, slots, fresh), plans[i]):
            buf.copy_(torch.tensor(values).to(buf.dtype))

    plan(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        prompt(window.clone(), state.clone())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    kept = window.clone(), state.clone()
    with torch.cuda.graph(graph):
        y = prompt(window, state)
    window.copy_(kept[0]), state.copy_(kept[1])
    for i in (0, 1, 2, 0):
        plan(i)
        w2, s2 = window.clone(), state.clone()
        graph.replay()
        want = prompt(w2, s2)
        assert torch.equal(torch.nan_to_num(y, 77.0), torch.nan_to_num(want, 77.0))
        assert torch.isnan(y).any() == (i == 2)
        assert torch.equal(window, w2) and torch.equal(state, s2)
