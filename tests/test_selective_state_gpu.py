"""Selective state operators on the GPU against the float64 oracle: short convolution and
scan over equal-length and packed sequences (lengths from none), training and prompts with
a pool, single tokens, odd widths, strides, groups, types, long batches that are cut into
pieces, refused slots, streams and captured graphs, and the mixer that runs them together.

Tolerances, in units of eps = 2^-24 times the same sums over absolute values (the oracle's
``absolute``), which bound every partial sum:

* convolution: K + 1 products and sums, the sigmoid (special-function exponential, 2^-22
  relative = 4 eps, of an argument that is off by |pre| eps; reciprocal 2 eps; four more
  roundings): (K + 12 + 2 |pre|) eps; 64 eps holds it for K <= 8 and |pre| <= 20.
* scan: every step rounds the state once, and its pole is off by 4 eps (special-function
  exponential) plus 4 eps |d A| (step, scaled A and their product); with |d A| exp(-|d A|)
  < 1/2 that is at most 4 + 2 + 1 eps per step of memory, on states whose absolute sums
  hold every term. Forward: (8 len + 64) eps. The adjoint has the same chain on top of the
  forward's: (16 len + 128) eps. Sums over rows or channels add at most their length.
* a result stored in bf16: half a step more, 2^-8 relative.
"""
from __future__ import annotations

import pytest
import torch

from oracle import selective_state as oss
from tests.parity import cuda, gen, randn

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24
HALF = {torch.float32: EPS, torch.bfloat16: 2.0 ** -8}


def _near(got, want, size, units, dtype, what):
    got = got.detach().double().cpu().reshape(want.shape)
    tol = units * EPS * size + HALF[dtype] * want.abs()
    if dtype == torch.bfloat16:
        tol = tol + 2.0 ** -126  # results that flush to zero
    # Steps below zero (no softplus) let a state grow: where the terms' sum passes 2^100 a partial
    # sum may pass what fp32 holds (2^128), and there is nothing to compare.
    over = torch.where(size < 2.0 ** 100, (got - want).abs() - tol, torch.zeros_like(want))
    assert bool((over <= 0).all()), f"{what}: over by {over.max().item():.3e} at {int(over.argmax())}, " \
        f"max error {(got - want).abs().max().item():.3e} of {want.abs().max().item():.3e}"


def _seqs(kind):
    """(offsets, rows) of a named batch."""
    lens = {"one": [1], "short": [3, 1, 2], "even": [21, 21, 21], "ragged": [0, 5, 0, 0, 33, 1, 70, 0, 17, 2, 0],
            "long": [300], "many": [1 + i * 7 % 40 for i in range(37)]}[kind]
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu, cu[-1] + (0 if kind in ("one", "even", "long") else 3)


def _batched(kind, t):
    """Equal-length kinds as (S, L, ...) without offsets, the others packed."""
    cu, _ = _seqs(kind)
    if kind in ("one", "even", "long"):
        return t.reshape((len(cu) - 1, cu[1]) + tuple(t.shape[1:])), None
    return t, torch.tensor(cu, dtype=torch.int32, device=cuda())


def _strided(t, pad):
    """t on the GPU as the middle of wider rows (pad elements on each side)."""
    wide = torch.full((t.shape[0], t[0].numel() + 2 * pad), float("nan"), dtype=t.dtype, device=cuda())
    wide[:, pad:pad + t[0].numel()] = t.reshape(t.shape[0], -1).to(wide.device)
    return wide[:, pad:pad + t[0].numel()].unflatten(-1, tuple(t.shape[1:]))


@pytest.mark.parametrize("kind", ["one", "short", "even", "ragged", "long", "many"])
@pytest.mark.parametrize("C,K,pad", [(1, 1, 0), (8, 4, 8), (7, 2, 3), (64, 3, 0), (136, 5, 8), (130, 8, 1), (520, 4, 0)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_conv_training(kind, C, K, pad, dtype):
    from semambaxlinoss_b200.selective_state import short_conv

    cu, rows = _seqs(kind)
    g = gen(C * 100 + K)
    x, dy = randn((rows, C), g).to(dtype), randn((rows, C), g).to(dtype)
    w, b = randn((C, K), g, scale=0.5).float(), randn((C,), g).float()
    silu = "silu" if K != 3 else None
    xd, cud = _batched(kind, _strided(x, pad))
    xd = xd.requires_grad_()
    wd, bd = w.to(cuda()).requires_grad_(), b.to(cuda()).requires_grad_()
    y = short_conv(xd, wd, bd, activation=silu, cu_seqlens=cud)
    dx, dw, db = torch.autograd.grad(y, (xd, wd, bd), _batched(kind, dy.to(cuda()))[0])
    args = [t.double() for t in (x, w, b)]
    out = oss.conv(*args, cu, silu is not None, dy=dy.double())
    size = oss.conv(*[t.abs() for t in args], cu, False, dy=dy.double().abs())
    assert y.shape == xd.shape and y.dtype == dtype and dx.dtype == dtype
    _near(y, out["y"], size["y"], 64, dtype, "y")
    # dpre = dy (s + pre s (1 - s)): |silu'| < 1.1, its error 16 eps (1 + |pre|) with |pre| <= size["y"].
    grow = 1.1 + size["y"].amax()
    _near(dx, out["dx"], size["dx"] * grow, 64, dtype, "dx")
    _near(dw, out["dw"], size["aw"] * grow, 64 + min(rows, 64) + 64, torch.float32, "dw")
    _near(db, out["db"], size["ab"] * grow, 64 + min(rows, 64) + 64, torch.float32, "db")
    assert not y.reshape(rows, C)[cu[-1]:].any() and not dx.reshape(rows, C)[cu[-1]:].any()


def _pool(S, shape, g, dtype):
    """Pool of S + 2 entries, shuffled slots (one sequence without), some sequences fresh."""
    pool = randn((S + 2,) + shape, g).to(dtype)
    slots = torch.randperm(S + 2, generator=g)[:S].to(torch.int32)
    if S > 2:
        slots[1] = -1
    fresh = torch.rand(S, generator=g) < 0.4
    start = [None if slots[s] < 0 or fresh[s] else pool[slots[s]].double() for s in range(S)]
    return pool, slots, fresh, start


@pytest.mark.parametrize("kind", ["one", "short", "even", "ragged", "long", "many"])
@pytest.mark.parametrize("C,K", [(8, 4), (7, 2), (136, 5), (64, 8), (256, 3)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_conv_prompts(kind, C, K, dtype):
    from semambaxlinoss_b200.selective_state import short_conv

    cu, rows = _seqs(kind)
    g = gen(C + 7 * K)
    S = len(cu) - 1
    x, w = randn((rows, C), g).to(dtype), randn((C, K), g, scale=0.5).float()
    pool, slots, fresh, start = _pool(S, (K - 1, C), g, dtype)
    xd, cud = _batched(kind, x.to(cuda()))
    pd = pool.to(cuda())
    y = short_conv(xd, w.view(C, 1, K).to(cuda()), None, cu_seqlens=cud, state=pd, slots=slots.to(cuda()),
                   fresh=fresh.to(cuda()))
    out = oss.conv(x.double(), w.double(), None, cu, windows=start)
    size = oss.conv(x.double().abs(), w.double().abs(), None, cu, False,
                    windows=[None if v is None else v.abs() for v in start])
    _near(y, out["y"], size["y"], 64, dtype, "y")
    want = pool.clone()
    for s in range(S):
        if slots[s] >= 0:
            want[slots[s]] = out["windows"][s].to(dtype)
    assert torch.equal(pd.cpu(), want)


def _scan_problem(rows, ch, N, G, g, dtype, dt_dtype=None):
    t = {"x": randn((rows, ch), g), "dt": randn((rows, ch), g, scale=0.7), "B": randn((rows, G, N), g),
         "C": randn((rows, G, N), g), "z": randn((rows, ch), g)}
    t = {k: v.to(dtype) for k, v in t.items()}
    t["dt"] = t["dt"].to(dt_dtype or dtype)
    t["A"] = -torch.exp(randn((ch, N), g, scale=0.7)).float()
    t["D"], t["dt_bias"] = randn((ch,), g).float(), (randn((ch,), g) - 2.0).float()
    return t


SCAN = [  # channels, modes, groups, pad, z, D and dt_bias, softplus
    (1, 1, 1, 0, True, True, True), (64, 16, 1, 0, True, True, True), (65, 16, 1, 3, True, False, True),
    (24, 3, 2, 1, False, True, False), (40, 8, 1, 8, True, True, True), (200, 4, 2, 0, True, True, True),
    (36, 20, 3, 0, False, False, True), (16, 64, 1, 2, True, True, True), (12, 128, 2, 0, True, True, True),
    (10, 33, 1, 0, True, True, True)]


@pytest.mark.parametrize("kind", ["one", "short", "even", "ragged", "long"])
@pytest.mark.parametrize("ch,N,G,pad,gate,extra,softplus", SCAN)
@pytest.mark.parametrize("dtype,dtt", [(torch.float32, None), (torch.bfloat16, None), (torch.bfloat16, torch.float32)])
def test_scan_training(kind, ch, N, G, pad, gate, extra, softplus, dtype, dtt):
    from semambaxlinoss_b200.selective_state import selective_state_scan

    cu, rows = _seqs(kind)
    g = gen(ch * 1000 + N)
    t = _scan_problem(rows, ch, N, G, g, dtype, dtt)
    if not softplus:
        t["dt"] = t["dt"].abs() * 0.3
    if not gate:
        t["z"] = None
    if not extra:
        t["D"] = t["dt_bias"] = None
    dy = randn((rows, ch), g).to(dtype)
    lead = ("x", "dt", "B", "C", "z")
    v = {k: None if t[k] is None else (_batched(kind, _strided(t[k], pad))[0] if k in lead else t[k].to(cuda()))
         for k in t}
    cud = _batched(kind, t["x"])[1]
    v = {k: None if u is None else u.requires_grad_() for k, u in v.items()}
    if G == 1 and not gate:
        v["B"], v["C"] = v["B"].squeeze(-2), v["C"].squeeze(-2)
    y = selective_state_scan(v["x"], v["dt"], v["A"], v["B"], v["C"], v["D"], v["z"], v["dt_bias"], softplus, cud)
    names = [k for k in v if v[k] is not None]
    grads = dict(zip(names, torch.autograd.grad(y, [v[k] for k in names], _batched(kind, dy.to(cuda()))[0])))
    d = {k: None if u is None else u.double() for k, u in t.items()}
    args = (d["x"], d["dt"], d["A"], d["B"], d["C"], cu, d["D"], d["z"], d["dt_bias"], softplus)
    out, size = oss.scan(*args, dy=dy.double()), oss.scan(*args, dy=dy.double(), absolute=True)
    longest = max(b - a for a, b in zip(cu[:-1], cu[1:]))
    assert y.shape == v["x"].shape and y.dtype == dtype
    _near(y, out["y"], size["y"], 8 * longest + 64, dtype, "y")
    units = 16 * longest + 128
    for k in names:
        got = grads[k]
        assert got.shape == v[k].shape and got.dtype == v[k].dtype
        n = units + (ch if k in ("B", "C") else rows if k in ("A", "D", "dt_bias") else 0)
        # dz is made from v as it was stored: half a step of dtype more.
        more = HALF[dtype] * size["dz"] / EPS if k == "z" else 0
        _near(got, out["d" + k], (size["d" + k] * n + more), 1, got.dtype, "d" + k)


@pytest.mark.parametrize("kind", ["one", "short", "even", "ragged", "long", "many"])
@pytest.mark.parametrize("ch,N,G", [(64, 16, 1), (24, 3, 2), (12, 128, 2), (33, 20, 1)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scan_prompts(kind, ch, N, G, dtype):
    from semambaxlinoss_b200.selective_state import selective_state_scan

    cu, rows = _seqs(kind)
    g = gen(ch + N)
    S = len(cu) - 1
    t = _scan_problem(rows, ch, N, G, g, dtype)
    pool, slots, fresh, start = _pool(S, (ch, N), g, torch.float32)
    v = {k: (_batched(kind, u.to(cuda()))[0] if k in ("x", "dt", "B", "C", "z") else u.to(cuda())) for k, u in t.items()}
    pd = pool.to(cuda())
    y = selective_state_scan(v["x"], v["dt"], v["A"], v["B"], v["C"], v["D"], v["z"], v["dt_bias"],
                             cu_seqlens=_batched(kind, t["x"])[1], state=pd, slots=slots.to(cuda()), fresh=fresh.to(cuda()))
    d = {k: u.double() for k, u in t.items()}
    args = (d["x"], d["dt"], d["A"], d["B"], d["C"], cu, d["D"], d["z"], d["dt_bias"])
    out, size = oss.scan(*args, h0=start), oss.scan(*args, h0=start, absolute=True)
    units = 8 * max(b - a for a, b in zip(cu[:-1], cu[1:])) + 64
    _near(y, out["y"], size["y"], units, dtype, "y")
    pd = pd.cpu()
    for s in range(S):
        if slots[s] >= 0:
            _near(pd[slots[s]], out["h"][s], size["h"][s], units, torch.float32, f"state {s}")
    others = [i for i in range(S + 2) if i not in slots.tolist()]
    assert torch.equal(pd[others], pool[others])


def test_long_sequences_in_pieces_equal_whole_ones():
    """A lone long sequence is cut into pieces (forward and backward); beside hundreds of
    copies of itself it is not. Same values within both paths' rounding, and the states of
    the pieces' ends are those of prompts in two calls."""
    from semambaxlinoss_b200.selective_state import selective_state_scan

    g, L, ch, N, many = gen(5), 500, 96, 16, 900
    t = _scan_problem(L, ch, N, 1, g, torch.float32)
    t = {k: u.to(cuda()) for k, u in t.items()}
    dy = randn((L, ch), g).float().to(cuda())

    def run(copies):
        v = {k: (u.expand(copies, *u.shape).contiguous() if k in ("x", "dt", "B", "C", "z") else u.clone()).requires_grad_()
             for k, u in t.items()}
        y = selective_state_scan(v["x"], v["dt"], v["A"], v["B"], v["C"], v["D"], v["z"], v["dt_bias"])
        gr = torch.autograd.grad(y, [v[k] for k in ("x", "dt", "B", "C", "z")], dy.expand(copies, L, ch))
        return [u[0] for u in (y,) + gr]

    for p, q in zip(run(1), run(many)):
        assert (p - q).abs().max() <= (16 * L + 128) * EPS * 4 * q.abs().max()
    one, two = torch.zeros(1, ch, N, device=cuda()), torch.zeros(1, ch, N, device=cuda())

    def prompt(lo, hi, state):
        return selective_state_scan(*[t[k][None, lo:hi] if k in ("x", "dt", "B", "C") else t[k]
                                      for k in ("x", "dt", "A", "B", "C")], D=t["D"], z=t["z"][None, lo:hi],
                                    dt_bias=t["dt_bias"], state=state)

    whole = prompt(0, L, one)
    parts = torch.cat([prompt(0, 1, two), prompt(1, 203, two), prompt(203, 203, two), prompt(203, L, two)], 1)
    assert (whole - parts).abs().max() <= (8 * L + 64) * EPS * 4 * whole.abs().max()
    assert (one - two).abs().max() <= (8 * L + 64) * EPS * 4 * one.abs().max()


def test_a_long_prompt_among_short_ones():
    """A packed batch that fills the GPU with one sequence far longer than the others, which is
    then cut while they stay whole: outputs, states and gradients of every sequence are those
    of the sequence alone, within both ways' rounding; a refused slot and an absent one too."""
    from semambaxlinoss_b200.selective_state import selective_state_scan

    g, ch, N = gen(17), 520, 16
    lens = [3, 900, 1, 0] + [2 + i % 7 for i in range(50)]
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    rows, S = cu[-1] + 5, len(lens)
    t = {k: u.to(cuda()) for k, u in _scan_problem(rows, ch, N, 1, g, torch.float32).items()}
    cud = torch.tensor(cu, dtype=torch.int32, device=cuda())
    par = {k: t[k] for k in ("D", "dt_bias")}
    units = (16 * 900 + 128) * EPS * 4

    def run(sel, **kw):
        v = {k: t[k][sel].clone().requires_grad_() for k in ("x", "dt", "B", "C", "z")}
        y = selective_state_scan(v["x"], v["dt"], t["A"], v["B"], v["C"], z=v["z"], **par, **kw)
        return [y] + list(torch.autograd.grad(y, list(v.values()), torch.ones_like(y)))

    whole = run(slice(None), cu_seqlens=cud)
    pool = torch.randn(S + 1, ch, N, device=cuda())
    slots = torch.randperm(S + 1, generator=g)[:S].to(torch.int32)
    slots[0], slots[4] = -1, slots[1]  # no entry; the long prompt's entry again
    after = pool.clone()
    with torch.no_grad():
        y = selective_state_scan(t["x"], t["dt"], t["A"], t["B"], t["C"], z=t["z"], **par, cu_seqlens=cud, state=after,
                                 slots=slots.to(cuda()))
    assert torch.isnan(y[cu[4]:cu[5]]).all()
    for s in (0, 1, 2, 5, S - 1):
        sel = slice(cu[s], cu[s + 1])
        one = torch.tensor([0, lens[s]], dtype=torch.int32, device=cuda())
        for p, q in zip(whole, run(sel, cu_seqlens=one)):
            assert (p[sel] - q).abs().max() <= units * q.abs().max(), s
        state = pool[slots[s].clamp(min=0)][None].clone() if slots[s] >= 0 else torch.zeros(1, ch, N, device=cuda())
        with torch.no_grad():
            want = selective_state_scan(t["x"][sel], t["dt"][sel], t["A"], t["B"][sel], t["C"][sel], z=t["z"][sel], **par,
                                        cu_seqlens=one, state=state)
        assert (y[sel] - want).abs().max() <= units * want.abs().max(), s
        if slots[s] >= 0:
            assert (after[slots[s]] - state[0]).abs().max() <= units * state.abs().max(), s
    for e in [i for i in range(S + 1) if i not in slots.tolist()] + [int(slots[3])]:
        assert torch.equal(after[e], pool[e])
    assert not y[cu[-1]:].any() and not whole[1][cu[-1]:].any()


@pytest.mark.parametrize("S", [1, 5, 150])
@pytest.mark.parametrize("ch,N,G,K", [(8, 4, 1, 4), (65, 16, 1, 4), (24, 3, 2, 2), (12, 128, 2, 3), (520, 16, 1, 8)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_single_tokens(S, ch, N, G, K, dtype):
    from semambaxlinoss_b200.selective_state import selective_state_step, short_conv_step

    g = gen(S * ch)
    t = _scan_problem(S, ch, N, G, g, dtype)
    w, b = randn((ch, K), g).float(), randn((ch,), g).float()
    wins, slots, _, start = _pool(S, (K - 1, ch), g, dtype)
    start = [None if slots[s] < 0 else wins[slots[s]].double() for s in range(S)]
    wd, sd = wins.to(cuda()), slots.to(cuda())
    y = short_conv_step(_strided(t["x"], 8), wd, w.to(cuda()), b.to(cuda()), slots=sd)
    cu = list(range(S + 1))
    out = oss.conv(t["x"].double(), w.double(), b.double(), cu, windows=start)
    size = oss.conv(t["x"].double().abs(), w.double().abs(), b.double().abs(), cu, False,
                    windows=[None if v is None else v.abs() for v in start])
    _near(y, out["y"], size["y"], 64, dtype, "conv")
    for s in range(S):
        if slots[s] >= 0:
            wins[slots[s]] = out["windows"][s].to(dtype)
    assert torch.equal(wd.cpu(), wins)
    pool = randn((S + 2, ch, N), g).float()
    start = [None if slots[s] < 0 else pool[slots[s]].double() for s in range(S)]
    pd = pool.to(cuda())
    v = {k: u.to(cuda()) for k, u in t.items()}
    y = selective_state_step(v["x"], v["dt"], v["A"], v["B"], v["C"], pd, v["D"], v["z"], v["dt_bias"], slots=sd)
    d = {k: u.double() for k, u in t.items()}
    args = (d["x"], d["dt"], d["A"], d["B"], d["C"], cu, d["D"], d["z"], d["dt_bias"])
    out, size = oss.scan(*args, h0=start), oss.scan(*args, h0=start, absolute=True)
    _near(y, out["y"], size["y"], 72, dtype, "y")
    for s in range(S):
        if slots[s] >= 0:
            _near(pd.cpu()[slots[s]], out["h"][s], size["h"][s], 72, torch.float32, "state")
    others = [i for i in range(S + 2) if i not in slots.tolist()]
    assert torch.equal(pd.cpu()[others], pool[others])


def _ops(S, ch=40, N=16):
    """Prompts of 3 rows and single tokens through both operators: (name, call(x rows, slots) -> y, pool)."""
    from semambaxlinoss_b200.selective_state import (selective_state_scan, selective_state_step, short_conv,
                                                     short_conv_step)

    g = gen(9)
    t = {k: u.to(cuda()) for k, u in _scan_problem(3 * S, ch, N, 1, g, torch.float32).items()}
    w = randn((ch, 4), g).float().to(cuda())
    seq = {k: t[k].view(S, 3, *t[k].shape[1:]) for k in ("x", "dt", "B", "C", "z")}
    one = {k: seq[k][:, 0] for k in seq}
    return [
        ("conv", lambda p, s: short_conv(seq["x"], w, state=p, slots=s), (3, ch)),
        ("conv step", lambda p, s: short_conv_step(one["x"], p, w, slots=s), (3, ch)),
        ("scan", lambda p, s: selective_state_scan(seq["x"], seq["dt"], t["A"], seq["B"], seq["C"], t["D"], seq["z"],
                                                   state=p, slots=s), (ch, N)),
        ("scan step", lambda p, s: selective_state_step(one["x"], one["dt"], t["A"], one["B"], one["C"], p, t["D"],
                                                        one["z"], slots=s), (ch, N))]


def test_refused_and_absent_slots():
    """A slot behind the pool, and one that an earlier sequence has, give NaN and touch
    nothing; a negative one starts from zeros and leaves nothing; the others are as alone."""
    S = 6
    for name, call, shape in _ops(S):
        pool = torch.randn((S + 1,) + shape, device=cuda())
        good = torch.tensor([3, 0, 6, 1, 2, 5], dtype=torch.int32, device=cuda())
        p0 = pool.clone()
        want = call(p0, good)
        bad = torch.tensor([3, 7, 6, 3, -1, 2147483647], dtype=torch.int32, device=cuda())
        p1 = pool.clone()
        got = call(p1, bad)
        for s in (1, 3, 5):
            assert torch.isnan(got[s]).all(), name
        for s in (0, 2):
            assert torch.equal(got[s], want[s]) and torch.equal(p1[good[s]], p0[good[s]]), name
        for e in (0, 1, 2, 4, 5):
            assert torch.equal(p1[e], pool[e]), name
        zero = torch.zeros_like(pool)
        assert torch.equal(got[4], call(zero, good)[4]), name


def test_non_finite_rows_stay_in_their_sequence():
    from semambaxlinoss_b200.selective_state import selective_state_scan, short_conv

    g = gen(3)
    cu, ch = torch.tensor([0, 9, 20, 29], dtype=torch.int32, device=cuda()), 40
    t = {k: u.to(cuda()) for k, u in _scan_problem(32, ch, 16, 1, g, torch.float32).items()}
    w = torch.randn(ch, 4, device=cuda())

    def run(x):
        v = {k: u.detach().clone().requires_grad_() for k, u in dict(t, x=x, w=w).items()}
        u = short_conv(v["x"], v["w"], cu_seqlens=cu)
        y = selective_state_scan(u, v["dt"], v["A"], v["B"], v["C"], v["D"], v["z"], v["dt_bias"], cu_seqlens=cu)
        return [y.detach()] + list(torch.autograd.grad(y.sum(), [v["x"], v["dt"], v["z"]]))

    clean = run(t["x"])
    for value in (float("nan"), float("inf")):
        x = t["x"].clone()
        x[12, 3] = value  # second sequence
        x[30] = value     # behind the last sequence
        for p, q in zip(run(x), clean):
            assert torch.equal(p[:9], q[:9]) and torch.equal(p[20:], q[20:])
            assert torch.isfinite(p[9:20, :3]).all() and torch.isfinite(p[9:20, 4:]).all()


def test_steps_far_out():
    """Softplus at its ends: exact to 2 steps of fp32 from tiny steps to large ones, zero at
    -inf (the state stays as it is), NaN at NaN. One row per sequence with x = B = C = 1, A = 0
    and no entry state, so that y is the step itself."""
    from semambaxlinoss_b200.selective_state import selective_state_scan, selective_state_step

    v = torch.cat([torch.linspace(-30, 30, 997), torch.tensor([-100.0, -87.0, 20.0, 20.5, 88.0, 1e4, float("-inf"), float("nan")])])
    ch = v.numel()
    dt, one = v.to(cuda()).view(1, 1, ch), torch.ones(1, 1, ch, device=cuda())
    BC, A = torch.ones(1, 1, 1, device=cuda()), torch.zeros(ch, 1, device=cuda())
    want = torch.nn.functional.softplus(v.double())
    state = torch.zeros(1, ch, 1, device=cuda())
    for y in (selective_state_scan(one, dt, A, BC, BC), selective_state_step(one[0], dt[0], A, BC[0], BC[0], state)):
        y = y.reshape(-1).double().cpu()
        assert torch.isnan(y[-1])
        # 1e-7 of the series, 4 eps of the exponential, a few roundings; below exp(-87) fp32 flushes.
        assert ((y - want)[:-1].abs() <= 8 * EPS * want[:-1] + 2.0 ** -126).all()


@pytest.mark.parametrize("L", [1, 3, 16, 18])
def test_a_step_of_zero_keeps_the_state(L):
    """dt = -inf is a step of exactly zero: pole 1, no drive; the entry keeps its bits, at lengths
    that end inside a tile too (rows behind the end are steps of zero)."""
    from semambaxlinoss_b200.selective_state import selective_state_scan, selective_state_step

    ch, N = 70, 16
    A, BC = -torch.rand(ch, N, device=cuda()) * 20, torch.randn(2, L, N, device=cuda())
    x, dt = torch.randn(2, L, ch, device=cuda()), torch.full((2, L, ch), float("-inf"), device=cuda())
    state = torch.randn(2, ch, N, device=cuda())
    kept = state.clone()
    y = selective_state_scan(x, dt, A, BC, BC, state=state)
    assert torch.equal(state, kept) and torch.isfinite(y).all()
    selective_state_step(x[:, 0], dt[:, 0], A, BC[:, 0], BC[:, 0], state)
    assert torch.equal(state, kept)


@pytest.mark.parametrize("L", [1, 3, 18, 300])
def test_a_rate_of_minus_infinity_forgets(L):
    """A = -inf (its logarithm ran away) is a pole of zero: every mode holds its last drive, no
    NaN comes up at lengths that end inside a tile, and the gradients are those of a finite
    rate whose poles are zero too (1e30 with steps above 1e-3)."""
    from semambaxlinoss_b200.selective_state import selective_state_scan, selective_state_step

    g = gen(11)
    ch, N = 40, 16
    t = {k: u.to(cuda()) for k, u in _scan_problem(2 * L, ch, N, 1, g, torch.float32).items()}
    rows = {k: t[k].reshape(2, L, *t[k].shape[1:]) for k in ("x", "dt", "B", "C", "z")}
    rows["dt"] = rows["dt"].abs()

    def run(rate):
        A = t["A"].clone()
        A[3:9, 1::3] = rate
        state = torch.zeros(2, ch, N, device=cuda())
        with torch.no_grad():
            y = selective_state_scan(rows["x"], rows["dt"], A, rows["B"], rows["C"], t["D"], rows["z"], state=state)
            last = selective_state_step(*(rows[k][:, 0] for k in ("x", "dt")), A, rows["B"][:, 0], rows["C"][:, 0], state)
        v = {k: u.detach().clone().requires_grad_() for k, u in rows.items()}
        out = selective_state_scan(v["x"], v["dt"], A, v["B"], v["C"], t["D"], v["z"])
        return [y, state, last, out.detach()] + list(torch.autograd.grad(out.square().sum(), list(v.values())))

    for got, want in zip(run(float("-inf")), run(-1e30)):
        assert torch.isfinite(want).all() and torch.equal(got, want)


def test_bad_offsets_stay_inside():
    """Offsets that decrease, start below zero or reach behind the rows give some result
    without an access outside (they are clamped in the kernels)."""
    from semambaxlinoss_b200.selective_state import selective_state_scan, short_conv

    t = {k: u.to(cuda()) for k, u in _scan_problem(30, 16, 16, 1, gen(4), torch.float32).items()}
    for cu in ([-5, 10, 4, 99, 20], [30, 0, 0, 0, 0], [2147483647, -2147483648, 5, 5, 5], [40, 50, 60, 70, 80]):
        cud = torch.tensor(cu, dtype=torch.int32, device=cuda())
        v = {k: u.clone().requires_grad_() for k, u in t.items()}
        y = short_conv(v["x"], torch.ones(16, 4, device=cuda()), cu_seqlens=cud)
        y = selective_state_scan(y, v["dt"], v["A"], v["B"], v["C"], v["D"], v["z"], v["dt_bias"], cu_seqlens=cud)
        torch.autograd.grad(y.sum(), [v["x"]])
        state = torch.zeros(4, 16, 16, device=cuda())
        with torch.no_grad():
            selective_state_scan(*[t[k] for k in ("x", "dt", "A", "B", "C")], cu_seqlens=cud, state=state)
        torch.cuda.synchronize()


def test_offsets_past_32_bits():
    """Operands that are slices of rows 2^20 elements long: row 2500 begins behind element 2^31.
    The same values as with rows of their own, bit for bit."""
    from semambaxlinoss_b200.selective_state import selective_state_scan, short_conv

    rows, ch, N = 2600, 32, 16
    wide = torch.empty(rows, 1 << 20, dtype=torch.bfloat16, device=cuda())
    part = wide[:, -(3 * ch + 2 * N):]
    part.normal_()
    x, dt, z, B, C = part.split([ch, ch, ch, N, N], -1)
    A = -torch.rand(ch, N, device=cuda()) - 0.1
    w = torch.randn(ch, 4, device=cuda())
    cu = torch.tensor([0, 700, 2590], dtype=torch.int32, device=cuda())

    def run(x, dt, z, B, C):
        leaves = [t.detach().requires_grad_() for t in (x, dt, z, B, C)]
        u = short_conv(leaves[0], w, cu_seqlens=cu)
        y = selective_state_scan(u, leaves[1], A, leaves[3], leaves[4], z=leaves[2], cu_seqlens=cu)
        return [y] + list(torch.autograd.grad(y, leaves, torch.ones_like(y)))

    for p, q in zip(run(x, dt, z, B, C), run(*[t.contiguous() for t in (x, dt, z, B, C)])):
        assert torch.equal(p, q)


def test_no_sequences_and_no_rows():
    from semambaxlinoss_b200.selective_state import selective_state_scan, selective_state_step, short_conv

    dev, ch, N = cuda(), 16, 4
    none = torch.zeros(1, dtype=torch.int32, device=dev)
    A, w = -torch.rand(ch, N, device=dev), torch.rand(ch, 4, device=dev)
    for rows, cu in ((7, none), (0, none), (0, torch.zeros(4, dtype=torch.int32, device=dev))):
        x = torch.randn(rows, ch, device=dev, requires_grad=True)
        B = torch.randn(rows, N, device=dev, requires_grad=True)
        wl, Al = w.clone().requires_grad_(), A.clone().requires_grad_()
        y = selective_state_scan(short_conv(x, wl, cu_seqlens=cu), x, Al, B, B, z=x, cu_seqlens=cu)
        assert y.shape == (rows, ch) and not y.any()
        for gr in torch.autograd.grad(y, (x, wl, Al, B), torch.ones_like(y)):
            assert not gr.any()
    # Sequences of no rows leave their entries, or zeros if they are fresh.
    win, state = torch.ones(3, 3, ch, device=dev), torch.ones(3, ch, N, device=dev)
    x, B = torch.empty(0, ch, device=dev), torch.empty(0, N, device=dev)
    fresh = torch.tensor([False, True, False], device=dev)
    cu = torch.zeros(4, dtype=torch.int32, device=dev)
    short_conv(x, w, cu_seqlens=cu, state=win, fresh=fresh)
    selective_state_scan(x, x, A, B, B, cu_seqlens=cu, state=state, fresh=fresh)
    for pool in (win, state):
        assert bool((pool[[0, 2]] == 1).all()) and not pool[1].any()
    empty = torch.empty(0, 5, ch, device=dev)
    assert short_conv(empty, w).shape == empty.shape
    one = torch.empty(0, ch, device=dev)
    assert selective_state_step(one, one, A, one[:, :N], one[:, :N], state).shape == (0, ch)


def test_argument_checks():
    from semambaxlinoss_b200.selective_state import selective_state_scan, selective_state_step, short_conv

    dev = cuda()
    x, w, A, B = (torch.randn(s, device=dev) for s in ((2, 5, 8), (8, 4), (8, 4), (2, 5, 4)))
    cu = torch.zeros(3, dtype=torch.int32, device=dev)
    slots = torch.zeros(2, dtype=torch.int32, device=dev)
    win, state = torch.zeros(2, 3, 8, device=dev), torch.zeros(2, 8, 4, device=dev)
    conv_bad = [dict(x=x.half()), dict(x=x[0]), dict(cu_seqlens=cu), dict(x=x[0], cu_seqlens=cu.long()),
                dict(x=x[0], cu_seqlens=cu.cpu()), dict(weight=w[:4]), dict(weight=torch.randn(8, 9, device=dev)),
                dict(weight=w.cpu()), dict(bias=w[:, 0][:4]), dict(activation="relu"), dict(slots=slots),
                dict(state=win[:1]), dict(state=win.bfloat16()), dict(state=win.transpose(1, 2)), dict(state=win[:0], slots=slots),
                dict(state=win, slots=slots.long()), dict(state=win, slots=slots[:1]), dict(state=win, fresh=slots),
                dict(state=win, weight=w.clone().requires_grad_())]
    for bad in conv_bad:
        with pytest.raises(ValueError):
            short_conv(**{**dict(x=x, weight=w), **bad})
    scan_bad = [dict(x=x.half()), dict(dt=x[:, :4]), dict(dt=x.bfloat16()), dict(A=A[:4]), dict(A=A[:, :0]),
                dict(A=torch.randn(8, 129, device=dev)), dict(B=B.bfloat16()), dict(C=B[..., :3]), dict(B=B[0]),
                dict(B=B.view(2, 5, 1, 4)), dict(z=x.bfloat16()), dict(D=A[:, 0][:4]), dict(dt_bias=A[0]),
                dict(B=torch.randn(2, 5, 3, 4, device=dev), C=torch.randn(2, 5, 3, 4, device=dev)),
                dict(state=state.bfloat16()), dict(state=state[:1]), dict(state=state, A=A.clone().requires_grad_()),
                dict(fresh=torch.zeros(2, dtype=torch.bool, device=dev))]
    for bad in scan_bad:
        with pytest.raises(ValueError):
            selective_state_scan(**{**dict(x=x, dt=x, A=A, B=B, C=B), **bad})
    with pytest.raises(ValueError):
        selective_state_step(x, x, A, B, B, state)
    with pytest.raises(ValueError):
        selective_state_step(x[:, 0], x[:, 0], A, B[:, 0], B[:, 0], None)


def test_gradients_against_differences():
    """The operators' own outputs, moved along one direction of every operand: fp32 values
    of size 1 hold 2^-24 of it, so a step of 2^-7 shows the slope to about 2^-7 of itself
    squared (third derivatives) plus (8 len + 64) 2^-24 / 2^-7 of the sum's absolute size."""
    from semambaxlinoss_b200.selective_state import selective_state_scan, short_conv

    g, rows, ch, N = gen(11), 24, 40, 16
    cu = torch.tensor([0, 7, 7, 20], dtype=torch.int32, device=cuda())
    t = _scan_problem(rows, ch, N, 2, g, torch.float32)
    t |= {"w": randn((ch, 4), g).float(), "b": randn((ch,), g).float()}
    t = {k: u.to(cuda()) for k, u in t.items()}
    move = {k: randn(u.shape, g, scale=0.3).float().to(cuda()) for k, u in t.items()}
    weight = randn((rows, ch), g).float().to(cuda())

    def value(v):
        u = short_conv(v["x"], v["w"], v["b"], cu_seqlens=cu)
        return selective_state_scan(u, v["dt"], v["A"], v["B"], v["C"], v["D"], v["z"], v["dt_bias"], cu_seqlens=cu)

    leaves = {k: u.clone().requires_grad_() for k, u in t.items()}
    grads = torch.autograd.grad(value(leaves), list(leaves.values()), weight)
    slope = sum((p.double() * move[k].double()).sum() for p, k in zip(grads, leaves))
    size = sum((p.double() * move[k].double()).abs().sum() for p, k in zip(grads, leaves))
    h = 2.0 ** -7
    up, down = (value({k: t[k] + s * h * move[k] for k in t}).double() for s in (1, -1))
    diff = ((up - down) * weight).sum() / (2 * h)
    noise = (8 * 13 + 64) * EPS / h * 4 * (up.abs() * weight.abs()).sum()
    assert (diff - slope).abs() <= 4 * h * h * size + noise


def test_deterministic_streams_and_captured_graphs():
    """The same call twice gives the same bits; on a side stream too; a captured training
    pass and a captured decoding step give on replay what a plain call gives."""
    from semambaxlinoss_b200.selective_state import (selective_state_scan, selective_state_step, short_conv,
                                                     short_conv_step)

    g, S, L, ch, N = gen(13), 3, 130, 72, 16
    t = {k: u.to(cuda()) for k, u in _scan_problem(S * L, ch, N, 1, g, torch.bfloat16).items()}
    t = {k: (u.view(S, L, *u.shape[1:]) if k in ("x", "dt", "B", "C", "z") else u) for k, u in t.items()}
    t["w"] = torch.randn(ch, 4, device=cuda())
    dy = torch.randn(S, L, ch, device=cuda()).bfloat16()
    leaves = {k: u.detach().requires_grad_() for k, u in t.items()}

    def train():
        u = short_conv(leaves["x"], leaves["w"])
        y = selective_state_scan(u, *[leaves[k] for k in ("dt", "A", "B", "C", "D", "z", "dt_bias")])
        return [y.detach()] + list(torch.autograd.grad(y, list(leaves.values()), dy))

    win, state = torch.zeros(S, 3, ch, device=cuda(), dtype=torch.bfloat16), torch.zeros(S, ch, N, device=cuda())
    slots = torch.arange(S, dtype=torch.int32, device=cuda())
    one = {k: t[k][:, 0].contiguous() for k in ("x", "dt", "B", "C", "z")}

    def decode(w, s):
        u = short_conv_step(one["x"], w, t["w"], slots=slots)
        return selective_state_step(u, one["dt"], t["A"], one["B"], one["C"], s, t["D"], one["z"], t["dt_bias"], slots=slots)

    want = train()
    assert all(torch.equal(p, q) for p, q in zip(want, train()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = train()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    graph, graph2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = train()
    with torch.cuda.graph(graph2):
        tok = decode(win, state)
    with torch.no_grad():
        t["x"].copy_(torch.randn_like(t["x"]))
        one["x"].copy_(torch.randn_like(one["x"]))
    win.zero_()
    state.zero_()
    w2, s2 = win.clone(), state.clone()
    graph.replay()
    for _ in range(3):
        graph2.replay()
        want_tok = decode(w2, s2)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(train(), out))
    assert torch.equal(tok, want_tok) and torch.equal(win, w2) and torch.equal(state, s2)


# -- the operators together: mixer, block, factory ----------------------------------------------


def _block(dtype=torch.float32, **cfg):
    from semambaxlinoss_b200.mamba_block import create_block

    torch.manual_seed(0)
    block = create_block(32, dict({"ssm": "selective_state", "d_state": 16, "d_conv": 4, "expand": 2}, **cfg),
                         rms_norm=False, fused_add_norm=True)
    with torch.no_grad():
        for p in block.parameters():
            p.add_(torch.randn(p.shape) * 0.05)
    return block.to(cuda(), dtype)


def _block_reference(p, x, residual, cu):
    """Pre-norm block with the selective state mixer on packed rows, float64."""
    s = x + residual
    h = torch.nn.functional.layer_norm(s, (32,), p["norm.weight"], p["norm.bias"])
    xz = h @ p["mixer.in_proj.weight"].t()
    u, z = xz.chunk(2, -1)
    u = oss.conv(u, p["mixer.conv1d.weight"][:, 0], p["mixer.conv1d.bias"], cu)["y"]
    rows = u @ p["mixer.x_proj.weight"].t()
    dt = rows[:, :2] @ p["mixer.dt_proj.weight"].t()
    y = oss.scan(u, dt, -torch.exp(p["mixer.A_log"]), rows[:, None, 2:18], rows[:, None, 18:], cu, p["mixer.D"], z,
                 p["mixer.dt_proj.bias"])["y"]
    return y @ p["mixer.out_proj.weight"].t(), s


def test_block_training_matches_reference():
    """create_block(ssm selective_state, layer norm): output, residual and every gradient of the
    fused add + norm, projections, convolution and scan as one block. fp32 with GEMMs that
    sum up to 64 terms; errors of the inner results enter through a few products each: 1e-4
    of the largest value, the repository's bound for fp32 layers."""
    block = _block()
    g, cu = gen(21), [0, 19, 20, 41]
    x, r = randn((41, 32), g), randn((41, 32), g)
    dy, ds = randn((41, 32), g), randn((41, 32), g)
    params = {k: p.detach().double().cpu().requires_grad_() for k, p in block.named_parameters()}
    x64, r64 = x.clone().requires_grad_(), r.clone().requires_grad_()
    y64, s64 = _block_reference(params, x64, r64, cu)
    want = torch.autograd.grad((y64 * dy).sum() + (s64 * ds).sum(), [x64, r64] + list(params.values()))
    xd, rd = (t.float().to(cuda()).requires_grad_() for t in (x, r))
    y, s = block(xd, rd, cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=cuda()))
    got = torch.autograd.grad((y, s), [xd, rd] + list(block.parameters()), [t.float().to(cuda()) for t in (dy, ds)])
    for name, p, q in zip(["y", "s", "x", "r"] + list(params), (y, s) + got, (y64, s64) + want):
        err = (p.detach().double().cpu() - q.detach()).abs().max() / q.detach().abs().max()
        assert err <= 1e-4, (name, err)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompts_and_tokens_equal_the_whole_sequence(dtype):
    """Prompts of several lengths through a cache with shuffled slots, then token by token (one
    sequence of the batch idle for a while), against the block on whole sequences. fp32: the
    repository's 1e-4. bf16: the two ways round the same quantities at the same places
    (projections' outputs), but GEMMs of other shapes may round a value the other way, 2^-8
    of it; a state averages many: 2e-2, the repository's bound."""
    block = _block().to(dtype)
    mixer = block.mixer
    g, lens, new = gen(23), [9, 1, 14], 5
    x = randn((3, 20, 32), g).to(dtype).to(cuda())
    tol = 1e-4 if dtype == torch.float32 else 2e-2
    slots = torch.tensor([4, 0, 2], dtype=torch.int32, device=cuda())
    with torch.no_grad():
        whole = [block(x[i:i + 1, :n + new], torch.zeros_like(x[i:i + 1, :n + new]))[0][0] for i, n in enumerate(lens)]
        cache = mixer.allocate_cache(5)
        cache.window.normal_()
        cache.state.normal_()
        cu = torch.tensor([0, 9, 10, 24], dtype=torch.int32, device=cuda())
        packed = torch.cat([x[i, :n] for i, n in enumerate(lens)])
        y, _ = block(packed, torch.zeros_like(packed), cu_seqlens=cu, cache=cache, slots=slots,
                     fresh=torch.ones(3, dtype=torch.bool, device=cuda()))
        for i, n in enumerate(lens):
            ref = whole[i].double()
            assert (y[cu[i]:cu[i + 1]].double() - ref[:n]).abs().max() <= tol * ref.abs().max()
        pos = list(lens)
        for step in range(2 * new):
            # A padded batch of three rows: sequence 1 sits out every other call.
            act = [pos[i] < lens[i] + new and (i != 1 or step % 2 == 0) for i in range(3)]
            tok = torch.stack([x[i, min(pos[i], 19)] for i in range(3)])[:, None]
            idx = torch.tensor([int(slots[i]) if act[i] else -1 for i in range(3)], dtype=torch.int32, device=cuda())
            y, _ = block(tok, torch.zeros_like(tok), cache=cache, slots=idx)
            for i in range(3):
                if act[i]:
                    ref = whole[i].double()
                    assert (y[i, 0].double() - ref[pos[i]]).abs().max() <= tol * ref.abs().max(), (step, i)
                    pos[i] += 1
        assert pos == [n + new for n in lens]


@pytest.mark.parametrize("width,modes,taps,groups", [(24, 8, 1, 2), (15, 5, 8, 3), (33, 16, 2, 1)])
def test_mixer_widths_and_captured_tokens(width, modes, taps, groups):
    """One tap (no window to keep), many taps, groups, widths that leave rows unaligned: a prompt,
    then tokens from a replayed graph, against the whole sequence (fp32: the repository's 1e-4)."""
    from semambaxlinoss_b200.selective_state import SelectiveStateMixer

    torch.manual_seed(3)
    mixer = SelectiveStateMixer(width, modes, taps, 2, n_groups=groups).to(cuda())
    x = torch.randn(2, 12, width, device=cuda())
    slots = torch.tensor([2, 0], dtype=torch.int32, device=cuda())
    with torch.no_grad():
        whole = mixer(x)
        tol = 1e-4 * whole.abs().max()
        cache = mixer.allocate_cache(3)
        y = mixer(x[:, :7], cache=cache, slots=slots, fresh=torch.ones(2, dtype=torch.bool, device=cuda()))
        assert (y - whole[:, :7]).abs().max() <= tol
        token = x[:, 7].clone()
        kept = [t.clone() for t in (cache.window, cache.state)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            mixer.step(token, cache, slots)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = mixer.step(token, cache, slots)
        for t, k in zip((cache.window, cache.state), kept):
            t.copy_(k)
        for i in range(7, 12):
            token.copy_(x[:, i])
            graph.replay()
            assert (out - whole[:, i]).abs().max() <= tol


def test_bidirectional_block_and_autocast():
    """The factory's mixer inside MambaBlock: both directions, and bf16 autocast end to end."""
    from semambaxlinoss_b200.mamba_block import MambaBlock

    torch.manual_seed(3)
    m = MambaBlock(32, {"ssm": "selective_state", "d_state": 16, "d_conv": 4, "expand": 2}).to(cuda())
    x = torch.randn(2, 30, 32, device=cuda(), requires_grad=True)
    y = m(x)
    assert y.shape == (2, 30, 64)
    back = m.backward_blocks[0]
    flipped = back(torch.flip(x, [1]))
    torch.testing.assert_close(y[..., 32:], torch.flip(flipped[0] + flipped[1], [1]))
    with torch.autocast("cuda", dtype=torch.bfloat16):
        z = m(x)
    assert (z.double() - y.double()).abs().max() <= 2e-2 * y.abs().max()
    z.float().square().sum().backward()
    assert torch.isfinite(x.grad).all() and all(torch.isfinite(p.grad).all() for p in m.parameters())
