"""Gated recurrence on the GPU against the float64 oracle: equal-length and packed sequences
(lengths from none to several groups of tiles), training and prompts with a pool, single tokens, odd
widths, strides, types, refused slots, streams and captured graphs, and the mixer and block that run
it together with the convolution and the feed-forward half.

Tolerances, in units of eps = 2^-24 times the same sums over absolute values (the oracle's
``absolute``), which bound every partial sum. With |r + r_bias|, |i + i_bias| <= 8:

* a gate: exponential 4 eps of an argument 8 + 1 eps off, reciprocal 2, sum 1: 16 eps.
* la = -speed rho: 16 + softplus and products 8: 24 eps of |la|. The decay: 4 eps (far) or its
  rounding (near), and 26 |la| eps; |la| exp(-|la|) < 1/2, so what the las of a path of any length
  do to it is at most 13 eps, the rest at most 4 eps per step.
* gain: 1 - a^2 is 30 eps off (near: series and product on top of la's 24; far: 2 (4 + 26 / 2 eps) a^2
  where 1 - a^2 >= 1/2), its root half of that and 4 of the special function: 20 eps. Input: 40 eps.
* state: 4 + 1 roundings per step, and once more the same for the folded maps: (10 len + 64) eps;
  the gate silu(z) 20 eps: (10 len + 96) eps for y.
* gradients: the adjoint has the chain of the state again, dla multiplies both and 1 / gain:
  (24 len + 256) eps. Sums over rows add at most their number.
* a result stored in bf16: half a step more, 2^-8 relative.
"""
from __future__ import annotations

import pytest
import torch

from oracle import gated_lru as ogl
from tests.parity import cuda, gen, randn

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24
HALF = {torch.float32: EPS, torch.bfloat16: 2.0 ** -8}
BATCHES = {
    "one": [1], "short": [3, 1, 2], "even": [21, 21, 21], "tile": [64, 64], "over": [65, 65, 65],
    "ragged": [0, 5, 0, 0, 33, 1, 170, 0, 64, 2, 0], "long": [1100], "groups": [1024, 0, 2100, 63, 65, 1025],
    "many": [1 + i * 7 % 90 for i in range(37)],
}
WHOLE = ("one", "even", "tile", "over", "long")


def _near(got, want, size, units, dtype, what):
    got = got.detach().double().cpu().reshape(want.shape)
    tol = units * EPS * size + HALF[dtype] * want.abs() + 2.0 ** -126
    over = (got - want).abs() - tol
    assert bool((over <= 0).all()), f"{what}: over by {over.max().item():.3e} at {int(over.argmax())}, " \
        f"max error {(got - want).abs().max().item():.3e} of {want.abs().max().item():.3e}"


def _seqs(kind):
    cu = [0]
    for n in BATCHES[kind]:
        cu.append(cu[-1] + n)
    return cu, cu[-1] + (0 if kind in WHOLE else 3)


def _batched(kind, t):
    """Equal-length kinds as (S, L, ...) without offsets, the others packed."""
    cu, _ = _seqs(kind)
    if kind in WHOLE:
        return t.reshape((len(cu) - 1, cu[1]) + tuple(t.shape[1:])), None
    return t, torch.tensor(cu, dtype=torch.int32, device=cuda())


def _strided(t, pad):
    """t on the GPU as the middle of wider rows (pad elements on each side)."""
    wide = torch.full((t.shape[0], t.shape[1] + 2 * pad), float("nan"), dtype=t.dtype, device=cuda())
    wide[:, pad:pad + t.shape[1]] = t.to(wide.device)
    return wide[:, pad:pad + t.shape[1]]


def _operands(rows, C, dtype, g, fast=False):
    """(x, r, i, z) rows and (rate, r_bias, i_bias); ``fast``: decays far below 1 in some channels."""
    x, r, i, z = (randn((rows, C), g).to(dtype) for _ in range(4))
    r, i = r.clamp(-6, 6), i.clamp(-6, 6)
    rate = torch.rand(C, generator=g, dtype=torch.float64) * 5 - (5 if fast else 9)
    rate, rb, ib = rate.float(), randn((C,), g, scale=0.5).clamp(-2, 2).float(), randn((C,), g, scale=0.5).clamp(-2, 2).float()
    return [x, r, i, z], [rate, rb, ib]


def _oracle(rows, params, cu, h0=None, dy=None, gated=True, biased=True):
    x, r, i, z = (t.double() for t in rows)
    rate, rb, ib = (t.double() for t in params)
    kw = dict(z=z if gated else None, r_bias=rb if biased else None, i_bias=ib if biased else None, h0=h0, dy=dy)
    left = ogl.parts(r, i, rate, kw["r_bias"], kw["i_bias"])[4]
    assert not ((left / ogl.LEAST - 1).abs() < 1e-4).any()  # the border of the gain's gradient
    return (ogl.scan(x, r, i, rate, cu, **kw), ogl.scan(x, r, i, rate, cu, absolute=True, **kw))


@pytest.mark.parametrize("kind", list(BATCHES))
@pytest.mark.parametrize("C,pad,gated", [(1, 0, True), (7, 3, True), (64, 8, True), (130, 1, False), (136, 8, True),
                                         (72, 0, False)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_training(kind, C, pad, gated, dtype):
    from semambaxlinoss_b200.gated_lru import gated_lru_scan

    cu, rows = _seqs(kind)
    g = gen(C * 10 + pad)
    tok, par = _operands(rows, C, dtype, g, fast=C % 8 == 0)
    dy = randn((rows, C), g).to(dtype)
    biased = C != 72
    want, size = _oracle(tok, par, cu, dy=dy.double(), gated=gated, biased=biased)
    dev, cud = [], None
    for t in tok:
        t, cud = _batched(kind, _strided(t, pad))
        dev.append(t.requires_grad_())
    pd = [p.to(cuda()).requires_grad_() for p in par]
    kw = {"r_bias": pd[1], "i_bias": pd[2]} if biased else {}
    y = gated_lru_scan(dev[0], dev[1], dev[2], pd[0], z=dev[3] if gated else None, cu_seqlens=cud, **kw)
    ins = dev[:4 if gated else 3] + (pd if biased else pd[:1])
    names = ["dx", "dr", "di", "dz"][:4 if gated else 3] + ["drate", "dr_bias", "di_bias"][:3 if biased else 1]
    grads = torch.autograd.grad(y, ins, _batched(kind, dy.to(cuda()))[0])
    n = max(BATCHES[kind])
    assert y.shape == dev[0].shape and y.dtype == dtype
    _near(y, want["y"], size["y"], 10 * n + 96, dtype, "y")
    for name, got in zip(names, grads):
        whole = name in ("drate", "dr_bias", "di_bias")
        _near(got, want[name], size[name], 24 * n + 256 + (rows if whole else 0), torch.float32 if whole else dtype, name)
    for t in (y,) + tuple(grads[:4 if gated else 3]):
        assert not t.reshape(rows, C)[cu[-1]:].any()


def _pool(S, C, g):
    """Pool of S + 2 entries, shuffled slots (one sequence without), some sequences fresh."""
    pool = randn((S + 2, C), g).float()
    slots = torch.randperm(S + 2, generator=g)[:S].to(torch.int32)
    if S > 2:
        slots[1] = -1
    fresh = torch.rand(S, generator=g) < 0.4
    start = [None if slots[s] < 0 or fresh[s] else pool[slots[s]].double() for s in range(S)]
    return pool, slots, fresh, start


@pytest.mark.parametrize("kind", list(BATCHES))
@pytest.mark.parametrize("C,pad", [(1, 0), (7, 2), (136, 8), (64, 0), (257, 0)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompts(kind, C, pad, dtype):
    from semambaxlinoss_b200.gated_lru import gated_lru_scan

    cu, rows = _seqs(kind)
    g = gen(C + 5)
    S = len(cu) - 1
    tok, par = _operands(rows, C, dtype, g)
    pool, slots, fresh, start = _pool(S, C, g)
    want, size = _oracle(tok, par, cu, h0=start)
    dev, cud = [], None
    for t in tok:
        t, cud = _batched(kind, _strided(t, pad))
        dev.append(t)
    pd = [p.to(cuda()) for p in par]
    state = pool.to(cuda())
    y = gated_lru_scan(dev[0], dev[1], dev[2], pd[0], z=dev[3], r_bias=pd[1], i_bias=pd[2], cu_seqlens=cud,
                       state=state, slots=slots.to(cuda()), fresh=fresh.to(cuda()))
    n = max(BATCHES[kind])
    _near(y, want["y"], size["y"], 10 * n + 96, dtype, "y")
    after = pool.double()
    left = pool.double().abs()
    for s in range(S):
        if slots[s] >= 0:
            after[slots[s]], left[slots[s]] = want["h"][s], size["h"][s]
    _near(state, after, left, 10 * n + 96, torch.float32, "state")
    untouched = [e for e in range(S + 2) if e not in slots.tolist()]
    assert torch.equal(state[untouched].cpu(), pool[untouched])


@pytest.mark.parametrize("S,C,pad", [(1, 1, 0), (1, 2048, 0), (5, 7, 3), (33, 520, 8), (9, 130, 1), (200, 64, 0)])
@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_step(S, C, pad, gated, dtype):
    from semambaxlinoss_b200.gated_lru import gated_lru_step

    g = gen(S + C)
    tok, par = _operands(S, C, dtype, g, fast=True)
    pool, slots, _, _ = _pool(S, C, g)
    start = [None if slots[s] < 0 else pool[slots[s]].double() for s in range(S)]
    want, size = _oracle(tok, par, list(range(S + 1)), h0=start, gated=gated)
    dev, pd = [_strided(t, pad) for t in tok], [p.to(cuda()) for p in par]
    state = pool.to(cuda())
    y = gated_lru_step(dev[0], dev[1], dev[2], pd[0], state, z=dev[3] if gated else None, r_bias=pd[1], i_bias=pd[2],
                       slots=slots.to(cuda()))
    _near(y, want["y"], size["y"], 106, dtype, "y")
    for s in range(S):
        if slots[s] >= 0:
            _near(state[slots[s]], want["h"][s], size["h"][s], 106, torch.float32, f"state {s}")


def test_extreme_gates():
    """Gates shut (the lowest value, -inf) and open (inf), decays of 1 and 0, sizes of inputs."""
    from semambaxlinoss_b200.gated_lru import gated_lru_scan

    low, inf = torch.finfo(torch.float32).min, float("inf")
    r = torch.tensor([[low, -inf, inf, 0.0, 3.4e38, -100.0]] * 3)
    i = torch.tensor([[0.0, 0.0, 1.0, low, -inf, inf]] * 3)
    x = torch.tensor([[1.0, 2.0, 3.0, 4.0, 5.0, 6.0]] * 3)
    rate = torch.tensor([0.0, 1.0, 100.0, -3.0, -200.0, 2.0])
    tok = [t.double() for t in (x, r, i)]
    dy = torch.ones_like(x)
    want = ogl.scan(*tok, rate.double(), [0, 3], dy=dy.double())
    d = [t.to(cuda()).unsqueeze(0).requires_grad_() for t in (x, r, i)]
    rd = rate.to(cuda()).requires_grad_()
    y = gated_lru_scan(d[0], d[1], d[2], rd)
    grads = torch.autograd.grad(y, d + [rd], dy.to(cuda()).unsqueeze(0))
    for got, name in zip((y,) + grads, ("y", "dx", "dr", "di", "drate")):
        got = got.double().cpu().reshape(want[name].shape)
        assert torch.isfinite(got).all(), name
        assert torch.allclose(got, want[name], rtol=1e-5, atol=1e-30), (name, got, want[name])


def test_gradients_against_differences():
    """Central differences in float64 of the oracle's y, in one random direction per operand."""
    from semambaxlinoss_b200.gated_lru import gated_lru_scan

    cu, rows, C = [0, 70, 75, 150], 150, 24
    g = gen(8)
    tok, par = _operands(rows, C, torch.float32, g)
    dy = randn((rows, C), g)
    vals = [t.double() for t in tok + par]
    order = ("x", "r", "i", "z", "rate", "r_bias", "i_bias")

    def loss(v):
        x, r, i, z, rate, rb, ib = v
        return (ogl.scan(x, r, i, rate, cu, z, rb, ib)["y"] * dy).sum()

    dev = [t.float().to(cuda()).requires_grad_() for t in vals]
    x, r, i, z, rate, rb, ib = dev
    y = gated_lru_scan(x, r, i, rate, z=z, r_bias=rb, i_bias=ib,
                       cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=cuda()))
    grads = torch.autograd.grad(y, dev, dy.float().to(cuda()))
    for k, name in enumerate(order):
        v = randn(tuple(vals[k].shape), g)
        eps = 1e-5
        up, down = list(vals), list(vals)
        up[k], down[k] = vals[k] + eps * v, vals[k] - eps * v
        diff = (loss(up) - loss(down)) / (2 * eps)
        got = (grads[k].double().cpu() * v).sum()
        assert abs(got - diff) <= 2e-4 * (grads[k].double().cpu() * v).abs().sum(), (name, got, diff)


def test_pieces_equal_whole_and_repeat():
    """A prompt cut anywhere leaves what the whole one leaves; results do not change from run to run."""
    from semambaxlinoss_b200.gated_lru import gated_lru_scan, gated_lru_step

    g = gen(11)
    rows, C = 2500, 96
    tok, par = _operands(rows, C, torch.float32, g)
    x, r, i, z = (t.to(cuda()) for t in tok)
    rate, rb, ib = (t.to(cuda()) for t in par)
    kw = dict(r_bias=rb, i_bias=ib)
    state = torch.zeros(1, C, device=cuda())
    whole = gated_lru_scan(x[None], r[None], i[None], rate, z=z[None], state=state, **kw)[0]
    for _ in range(5):
        again = torch.zeros(1, C, device=cuda())
        assert torch.equal(gated_lru_scan(x[None], r[None], i[None], rate, z=z[None], state=again, **kw)[0], whole)
        assert torch.equal(again, state)
    part, outs = torch.zeros(1, C, device=cuda()), []
    for lo, hi in ((0, 1), (1, 64), (64, 1088), (1088, 2499)):
        s = slice(lo, hi)
        outs.append(gated_lru_scan(x[None, s], r[None, s], i[None, s], rate, z=z[None, s], state=part, **kw)[0])
    outs.append(gated_lru_step(x[2499:], r[2499:], i[2499:], rate, part, z=z[2499:], **kw))
    assert torch.allclose(torch.cat(outs), whole, rtol=1e-4, atol=1e-5)
    assert torch.allclose(part, state, rtol=1e-4, atol=1e-5)


def test_refused_slots():
    """A slot behind the pool, and one used twice: NaN rows, entries untouched, the others as alone."""
    from semambaxlinoss_b200.gated_lru import gated_lru_scan, gated_lru_step

    g = gen(3)
    C, lens = 40, [3, 1200, 2, 5, 70]
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    tok, par = _operands(cu[-1], C, torch.float32, g)
    x, r, i, z = (t.to(cuda()) for t in tok)
    rate = par[0].to(cuda())
    slots = torch.tensor([2, 9, 2, -1, 0], dtype=torch.int32, device=cuda())
    pool = randn((4, C), g).float().to(cuda())
    state = pool.clone()
    y = gated_lru_scan(x, r, i, rate, z=z, cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=cuda()), state=state,
                       slots=slots)
    assert torch.isnan(y[cu[1]:cu[3]]).all()
    assert torch.isfinite(y[:cu[1]]).all() and torch.isfinite(y[cu[3]:]).all()
    alone = pool[2:3].clone()
    want = gated_lru_scan(x[None, :3], r[None, :3], i[None, :3], rate, z=z[None, :3], state=alone)
    assert torch.equal(y[:3], want[0]) and torch.equal(state[2], alone[0])
    assert torch.equal(state[[1, 3]], pool[[1, 3]])
    st = pool.clone()
    out = gated_lru_step(x[:5], r[:5], i[:5], rate, st, slots=slots)
    assert torch.isnan(out[[1, 2]]).all() and torch.isfinite(out[[0, 3, 4]]).all()
    assert torch.equal(st[[1, 3]], pool[[1, 3]])


def test_bad_offsets_stay_inside():
    """Offsets that decrease or leave the rows give wrong rows, end, and touch nothing else."""
    from semambaxlinoss_b200.gated_lru import gated_lru_scan

    g = gen(4)
    rows, C = 400, 64
    tok, par = _operands(rows, C, torch.float32, g)
    wide = [torch.cat([t, torch.zeros(64, C)]).to(cuda()) for t in tok]
    x, r, i, z = (t[:rows] for t in wide)
    rate = par[0].to(cuda())
    for cu in ([0, 300, 100, 400], [350, 20, 399, 5], [-5, 100, 9999, 12], [0, 2 ** 31 - 1, -2 ** 31, 400], [5, 5, 5, 5]):
        c = torch.tensor(cu, dtype=torch.int32, device=cuda())
        y = gated_lru_scan(x, r, i, rate, z=z, cu_seqlens=c, state=torch.zeros(3, C, device=cuda()))
        assert y.shape == x.shape
        v = [t.clone().requires_grad_() for t in (x, r, i, z)]
        y = gated_lru_scan(v[0], v[1], v[2], rate, z=v[3], cu_seqlens=c)
        torch.autograd.grad(y, v, torch.ones_like(y))
    torch.cuda.synchronize()


def test_refusals():
    from semambaxlinoss_b200.gated_lru import gated_lru_scan, gated_lru_step

    C = 8
    x, rate = torch.zeros(2, 5, C, device=cuda()), torch.zeros(C, device=cuda())
    state = torch.zeros(3, C, device=cuda())
    slots, fresh = torch.zeros(2, dtype=torch.int32, device=cuda()), torch.zeros(2, dtype=torch.bool, device=cuda())
    good = dict(x=x, r=x, i=x, rate=rate, z=x, r_bias=rate, i_bias=rate, state=state, slots=slots, fresh=fresh)
    gated_lru_scan(**good)
    for bad, what in ((dict(r=x[:, :4]), "r must"), (dict(i=x.to(torch.bfloat16)), "i must"), (dict(z=x.cpu()), "z must"),
                      (dict(rate=rate[:7]), "rate must"), (dict(rate=rate.double()), "rate must"),
                      (dict(r_bias=rate[:3]), "r_bias"), (dict(i_bias=rate.cpu()), "i_bias"), (dict(x=x.double()), "dtype"),
                      (dict(rate_scale=0.0), "rate_scale"), (dict(rate_scale=float("inf")), "rate_scale"),
                      (dict(state=state[:, :4]), "state"), (dict(state=state.to(torch.bfloat16)), "state"),
                      (dict(state=state[:0]), "no entries"), (dict(state=state[:1], slots=None), "entries"),
                      (dict(slots=slots.long()), "slots"), (dict(fresh=slots), "fresh"), (dict(state=None), "without a state"),
                      (dict(rate=rate.clone().requires_grad_()), "inference"), (dict(x=x[0]), "batch"),
                      (dict(cu_seqlens=slots), "packed"), (dict(x=x[0], cu_seqlens=slots.long()), "cu_seqlens")):
        with pytest.raises(ValueError, match=what):
            gated_lru_scan(**dict(good, **bad))
    row = x[:, 0].contiguous()
    step = dict(x=row, r=row, i=row, rate=rate, state=state, z=row, slots=slots)
    gated_lru_step(**step)
    for bad, what in ((dict(x=x), "sequences, channels"), (dict(state=None), "needed"), (dict(r=row[:1]), "r must"),
                      (dict(z=row.clone().requires_grad_()), "inference"), (dict(state=state[:, :7]), "state")):
        with pytest.raises(ValueError, match=what):
            gated_lru_step(**dict(step, **bad))
    import torch.autograd.forward_ad as fwad

    with fwad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        gated_lru_scan(fwad.make_dual(x, torch.ones_like(x)), x, x, rate)


def test_broadcast_operands():
    """Expanded gates and rates: gradients are summed over what they were expanded along."""
    from semambaxlinoss_b200.gated_lru import gated_lru_scan

    g = gen(17)
    S, L, C = 3, 70, 24
    x, dy = (randn((S, L, C), g).float().to(cuda()) for _ in range(2))
    r, i = randn((1, L, C), g).float().to(cuda()).requires_grad_(), randn((S, 1, C), g).float().to(cuda()).requires_grad_()
    rate = torch.full((1,), -4.0, device=cuda(), requires_grad=True)
    got = torch.autograd.grad(gated_lru_scan(x, r.expand(S, L, C), i.expand(S, L, C), rate.expand(C)), (r, i, rate), dy)
    full = [t.detach().expand(n).contiguous().requires_grad_() for t, n in ((r, (S, L, C)), (i, (S, L, C)), (rate, (C,)))]
    want = torch.autograd.grad(gated_lru_scan(x, *full), full, dy)
    assert torch.allclose(got[0], want[0].sum(0, keepdim=True), rtol=1e-5, atol=1e-6)
    assert torch.allclose(got[1], want[1].sum(1, keepdim=True), rtol=1e-5, atol=1e-6)
    assert torch.allclose(got[2], want[2].sum(0, keepdim=True), rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("C", [8, 24000])
def test_few_and_many_channel_tiles(C):
    """One channel tile that all CTAs share, and more of them than CTAs run at once: forward, state and
    gradients of packed sequences against the walked form of the same rows."""
    from semambaxlinoss_b200.gated_lru import gated_lru_scan

    g = torch.Generator(device="cuda").manual_seed(C)
    S, L = (2, 3000) if C == 8 else (3, 100)
    x, r, i, z, dy = (torch.randn(S, L, C, generator=g, device="cuda") for _ in range(5))
    rate = torch.rand(C, generator=g, device="cuda") * 4 - 8
    cu = torch.arange(S + 1, dtype=torch.int32, device="cuda") * L

    def run(packed):
        f = (lambda t: t.reshape(S * L, C)) if packed else (lambda t: t)
        v = [f(t).clone().requires_grad_() for t in (x, r, i, z)] + [rate.clone().requires_grad_()]
        y = gated_lru_scan(v[0], v[1], v[2], v[4], z=v[3], cu_seqlens=cu if packed else None)
        return [t.reshape(S, L, C) if t.dim() > 1 else t for t in (y,) + torch.autograd.grad(y, v, f(dy))]

    for a, b in zip(run(True), run(False)):
        assert torch.allclose(a, b, rtol=1e-4, atol=1e-4 * float(b.abs().max()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_saved_tensors_moved(dtype):
    """Operands whose rows are strided, kept elsewhere between the passes: they come back dense."""
    from semambaxlinoss_b200.gated_lru import gated_lru_scan

    rows, params = _operands(170, 40, dtype, gen(6))
    ins = [_strided(t, 8).requires_grad_() for t in rows] + [p.to(cuda()).requires_grad_() for p in params]
    dy = randn((170, 40), gen(7)).to(dtype).to(cuda())
    cu = torch.tensor([0, 70, 70, 165], dtype=torch.int32, device=cuda())

    def run():
        x, r, i, z, rate, rb, ib = ins
        return gated_lru_scan(x, r, i, rate, z=z, r_bias=rb, i_bias=ib, cu_seqlens=cu)

    want = torch.autograd.grad(run(), ins, dy)
    with torch.autograd.graph.save_on_cpu():
        y = run()
    got = torch.autograd.grad(y, ins, dy)
    assert all(torch.equal(p[:165], q[:165]) if p.dim() == 2 else torch.equal(p, q) for p, q in zip(got, want))


def test_empty_batches():
    from semambaxlinoss_b200.gated_lru import gated_lru_scan, gated_lru_step

    dev = cuda()
    C = 12
    rate = torch.zeros(C, device=dev, requires_grad=True)
    for shape in ((0, 5, C), (3, 0, C)):
        x = torch.zeros(shape, device=dev, requires_grad=True)
        y = gated_lru_scan(x, x, x, rate)
        dx, dr = torch.autograd.grad(y.sum(), (x, rate))
        assert y.shape == shape and dx.shape == shape and not dr.any()
    none = torch.zeros(1, dtype=torch.int32, device=dev)
    x = torch.ones(9, C, device=dev)
    assert not gated_lru_scan(x, x, x, rate.detach(), cu_seqlens=none).any()
    big = torch.ones(300, C, device=dev, requires_grad=True)
    y = gated_lru_scan(big, big, big, rate, cu_seqlens=none)
    dx, dr = torch.autograd.grad(y, (big, rate), torch.ones_like(y))
    assert not y.any() and not dx.any() and not dr.any()
    state = torch.ones(2, C, device=dev)
    fresh = torch.tensor([True, False], device=dev)
    empty = torch.zeros(0, C, device=dev)
    gated_lru_scan(empty, empty, empty, rate.detach(), cu_seqlens=torch.zeros(3, dtype=torch.int32, device=dev),
                   state=state, fresh=fresh)
    assert not state[0].any() and bool((state[1] == 1).all())
    assert gated_lru_step(empty, empty, empty, rate.detach(), state).shape == (0, C)


def test_streams_and_graphs():
    """On another stream, two calls at once, and captured: the results of the plain call."""
    from semambaxlinoss_b200.gated_lru import gated_lru_scan

    g = gen(21)
    lens = [700, 3, 1300, 64]
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    C = 200
    tok, par = _operands(cu[-1], C, torch.bfloat16, g)
    x, r, i, z = (t.to(cuda()) for t in tok)
    rate = par[0].to(cuda())
    c = torch.tensor(cu, dtype=torch.int32, device=cuda())
    state0 = randn((4, C), g).float().to(cuda())
    state = state0.clone()
    want = gated_lru_scan(x, r, i, rate, z=z, cu_seqlens=c, state=state)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            st = state0.clone()
            got.append((gated_lru_scan(x, r, i, rate, z=z, cu_seqlens=c, state=st), st))
    torch.cuda.synchronize()
    for y, st in got:
        assert torch.equal(y, want) and torch.equal(st, state)
    # Two graphs that share a pool of memory, replayed in turn, with other offsets the second time.
    pool, graphs = torch.cuda.graph_pool_handle(), []
    static, st = c.clone(), state0.clone()
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            y = gated_lru_scan(x, r, i, rate, z=z, cu_seqlens=static, state=st)
        graphs.append((graph, y))
    for graph, y in graphs:
        st.copy_(state0)
        graph.replay()
        assert torch.equal(y, want) and torch.equal(st, state)
    other = torch.tensor([0, 1, 65, 1500, cu[-1]], dtype=torch.int32, device=cuda())
    state2 = state0.clone()
    want2 = gated_lru_scan(x, r, i, rate, z=z, cu_seqlens=other, state=state2)
    static.copy_(other)
    st.copy_(state0)
    graphs[0][0].replay()
    assert torch.equal(graphs[0][1], want2) and torch.equal(st, state2)


def test_captured_training():
    """A training pass captured into a graph gives the eager pass's gradients."""
    from semambaxlinoss_b200.gated_lru import gated_lru_scan

    g = gen(22)
    rows, C = 500, 72
    tok, par = _operands(rows, C, torch.float32, g)
    vals = [t.to(cuda()) for t in tok] + [par[0].to(cuda())]
    dy = randn((1, rows, C), g).float().to(cuda())

    def step():
        v = [t.detach().requires_grad_() for t in vals]
        y = gated_lru_scan(v[0][None], v[1][None], v[2][None], v[4], z=v[3][None])
        return (y,) + torch.autograd.grad(y, v, dy)

    want = [t.detach().clone() for t in step()]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_far_offsets():
    """Rows whose element offsets pass 2^31."""
    from semambaxlinoss_b200.gated_lru import gated_lru_scan

    g = gen(23)
    rows, C, ld = 40, 64, 60_000_000
    tok, par = _operands(rows, C, torch.bfloat16, g)
    wide = torch.empty(rows * ld // 8 * 8, dtype=torch.bfloat16, device=cuda())
    x = wide.as_strided((rows, C), (ld, 1))
    x.copy_(tok[0])
    r, i, z = (t.to(cuda()) for t in tok[1:])
    rate = par[0].to(cuda())
    c = torch.tensor([0, rows], dtype=torch.int32, device=cuda())
    got = gated_lru_scan(x, r, i, rate, z=z, cu_seqlens=c)
    assert torch.equal(got, gated_lru_scan(tok[0].to(cuda()), r, i, rate, z=z, cu_seqlens=c))


def _mixer(C, dtype, seed=0, **kw):
    from semambaxlinoss_b200.gated_lru import GatedLruMixer

    torch.manual_seed(seed)
    return GatedLruMixer(C, **kw).to(cuda(), dtype)


@pytest.mark.parametrize("C,kw", [(48, {}), (33, {"gate_rank": 5, "expand": 1, "d_conv": 2})])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_mixer_forms_agree(C, kw, dtype):
    """Whole sequences, a packed prompt with a cache, and token by token."""
    m = _mixer(C, dtype, **kw)
    m.rate.data = m.rate.data.float()
    g = gen(31)
    lens = [9, 1, 140]
    xs = [randn((n, C), g).to(dtype).to(cuda()) for n in lens]
    tol = dict(rtol=1e-4, atol=1e-4) if dtype == torch.float32 else dict(rtol=5e-2, atol=5e-2)
    with torch.no_grad():
        whole = [m(x[None])[0] for x in xs]
        cache = m.allocate_cache(4, dtype=dtype)
        slots = torch.tensor([3, 0, 2], dtype=torch.int32, device=cuda())
        fresh = torch.ones(3, dtype=torch.bool, device=cuda())
        cut = [6, 1, 100]
        cu = torch.tensor([0, 6, 7, 107], dtype=torch.int32, device=cuda())
        y = m(torch.cat([x[:n] for x, n in zip(xs, cut)]), cu_seqlens=cu, cache=cache, slots=slots, fresh=fresh)
        for k, (lo, hi) in enumerate(((0, 6), (6, 7), (7, 107))):
            assert torch.allclose(y[lo:hi].float(), whole[k][:cut[k]].float(), **tol)
        for t in range(3):
            for k, s in ((0, 6 + t), (2, 100 + t)):
                out = m(xs[k][None, s:s + 1], cache=cache, slots=slots[k:k + 1])
                assert torch.allclose(out[0, 0].float(), whole[k][s].float(), **tol)


def test_mixer_trains():
    """Every parameter of a training pass gets a finite gradient, which a difference confirms."""
    m = _mixer(32, torch.float32, seed=5)
    g = gen(32)
    x = randn((2, 70, 32), g).float().to(cuda())
    dy = randn((2, 70, 32), g).float().to(cuda())
    (m(x) * dy).sum().backward()
    for name, p in m.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all() and p.grad.any(), name
        v = p.grad / p.grad.norm()
        h = 1e-2 if p.dim() > 1 else 1e-3
        with torch.no_grad():
            old = p.detach().clone()
            p.copy_(old + h * v)
            up = (m(x).double() * dy.double()).sum()
            p.copy_(old - h * v)
            down = (m(x).double() * dy.double()).sum()
            p.copy_(old)
        diff = float((up - down) / (2 * h))
        assert abs(diff - float(p.grad.norm())) <= 2e-2 * float(p.grad.norm()) + 2e-3, (name, diff, float(p.grad.norm()))
