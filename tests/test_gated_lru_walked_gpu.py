"""Gated recurrence of many sequences of equal lengths: a CTA walks a sequence tile after tile and its state
stays in registers (no links, so no workspace in front of the backward's partial sums, which is what says
that a case runs so). Against the float64 oracle in both types, with ragged last tiles, odd widths and
strides, without output gate and biases, as training and as prompts with a pool. Tolerances as in
test_gated_lru_gpu.py; sums over the rows of all sequences have one rounding each at most."""
from __future__ import annotations

import pytest
import torch

from oracle import gated_lru as ogl
from tests.parity import cuda, gen, randn
from tests.test_gated_lru_gpu import _near, _operands, _strided

pytestmark = pytest.mark.gpu
# (sequences, length, channels): two tiles and a row, whole tiles, a part of one, several channel tiles, long ones; a
# tile of the forward is 64 steps, of the backward 32.
SIZES = [(600, 65, 8), (593, 130, 7), (600, 128, 1), (300, 200, 40), (150, 97, 130), (20, 330, 960), (592, 33, 24)]


def _side_by_side(t, S, L):
    """(S L, C) rows as the (L, S C) rows of one sequence, which is how the oracle takes equal lengths at once."""
    return t.reshape(S, L, -1).transpose(0, 1).reshape(L, -1)


def _back(t, S, L):
    return t.reshape(L, S, -1).transpose(0, 1).reshape(S * L, -1)


def _oracle(tok, par, S, L, h0=None, dy=None, gated=True, biased=True):
    """The oracle's results and their sizes, in the rows' order; parameters' gradients summed over sequences."""
    x, r, i, z = (_side_by_side(t.double(), S, L) for t in tok)
    rate, rb, ib = (p.double().repeat(S) for p in par)
    kw = dict(z=z if gated else None, r_bias=rb if biased else None, i_bias=ib if biased else None,
              h0=None if h0 is None else [h0.reshape(-1)], dy=None if dy is None else _side_by_side(dy.double(), S, L))
    left = ogl.parts(r, i, rate, kw["r_bias"], kw["i_bias"])[4]
    assert not ((left / ogl.LEAST - 1).abs() < 1e-4).any()  # the border of the gain's gradient
    out = []
    for absolute in (False, True):
        got = ogl.scan(x, r, i, rate, [0, L], absolute=absolute, **kw)
        res = {k: _back(v, S, L) for k, v in got.items() if k in ("y", "dx", "dr", "di", "dz")}
        res |= {k: got[k].reshape(S, -1).sum(0) for k in ("drate", "dr_bias", "di_bias") if k in got}
        out.append(dict(res, h=got["h"][0].reshape(S, -1)))
    return out


def _is_walked(S, L, C, backward):
    from semambaxlinoss_b200.gated_lru import _sizes

    _, fwd, bwd = _sizes(S, S * L, L, C, False)
    return bwd == S * 3 * C * 4 if backward else fwd == 0


@pytest.mark.parametrize("S,L,C", SIZES)
@pytest.mark.parametrize("gated,biased,pad", [(True, True, 0), (False, True, 8), (True, False, 3)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_training(S, L, C, gated, biased, pad, dtype):
    from semambaxlinoss_b200.gated_lru import gated_lru_scan

    assert _is_walked(S, L, C, False) and _is_walked(S, L, C, True)
    g = gen(S + L + C)
    tok, par = _operands(S * L, C, dtype, g, fast=C % 8 == 0)
    dy = randn((S * L, C), g).to(dtype)
    want, size = _oracle(tok, par, S, L, dy=dy, gated=gated, biased=biased)
    dev = [_strided(t, pad).unflatten(0, (S, L)).requires_grad_() for t in tok]
    pd = [p.to(cuda()).requires_grad_() for p in par]
    kw = {"r_bias": pd[1], "i_bias": pd[2]} if biased else {}
    y = gated_lru_scan(dev[0], dev[1], dev[2], pd[0], z=dev[3] if gated else None, **kw)
    ins = dev[:4 if gated else 3] + (pd if biased else pd[:1])
    names = ["dx", "dr", "di", "dz"][:4 if gated else 3] + ["drate", "dr_bias", "di_bias"][:3 if biased else 1]
    grads = torch.autograd.grad(y, ins, dy.to(cuda()).reshape(y.shape))
    _near(y, want["y"], size["y"], 10 * L + 96, dtype, "y")
    for name, got in zip(names, grads):
        whole = name in ("drate", "dr_bias", "di_bias")
        _near(got, want[name], size[name], 24 * L + 256 + (S * L if whole else 0), torch.float32 if whole else dtype, name)


@pytest.mark.parametrize("S,L,C", SIZES)
@pytest.mark.parametrize("gated,pad", [(True, 0), (False, 5)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompts(S, L, C, gated, pad, dtype):
    """A pool with shuffled slots, sequences without one, fresh ones, and two that are refused."""
    from semambaxlinoss_b200.gated_lru import gated_lru_scan

    assert _is_walked(S, L, C, False)
    g = gen(S * L + C)
    tok, par = _operands(S * L, C, dtype, g)
    pool = randn((S + 2, C), g).float()
    slots = torch.randperm(S + 2, generator=g)[:S].to(torch.int32)
    slots[1], slots[5], slots[S - 1] = -1, slots[3], S + 2
    fresh = torch.rand(S, generator=g) < 0.4
    refused, none = [5, S - 1], 1
    h0 = pool[slots.long().clamp(0, S + 1)].double()
    h0[fresh], h0[none] = 0, 0
    want, size = _oracle(tok, par, S, L, h0=h0, gated=gated)
    dev = [_strided(t, pad).unflatten(0, (S, L)) for t in tok]
    pd, state = [p.to(cuda()) for p in par], pool.to(cuda())
    y = gated_lru_scan(dev[0], dev[1], dev[2], pd[0], z=dev[3] if gated else None, r_bias=pd[1], i_bias=pd[2], state=state,
                       slots=slots.to(cuda()), fresh=fresh.to(cuda()))
    assert torch.isnan(y[refused]).all()
    keep = [s for s in range(S) if s not in refused]

    def of(t):
        return t.reshape(S, L, C)[keep]

    _near(y[keep], of(want["y"]), of(size["y"]), 10 * L + 96, dtype, "y")
    after, left = pool.double(), pool.double().abs()
    for s in keep:
        if slots[s] >= 0:
            after[slots[s]], left[slots[s]] = want["h"][s], size["h"][s]
    _near(state, after, left, 10 * L + 96, torch.float32, "state")
    used = {int(slots[s]) for s in keep}
    untouched = [e for e in range(S + 2) if e not in used]
    assert torch.equal(state[untouched].cpu(), pool[untouched])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_repeats_and_graphs(dtype):
    """The same bits from run to run, from a prompt without a pool as from one with fresh sequences, and from a
    captured training pass."""
    from semambaxlinoss_b200.gated_lru import gated_lru_scan

    S, L, C = 300, 150, 40
    assert _is_walked(S, L, C, True)
    g = gen(9)
    tok, par = _operands(S * L, C, dtype, g)
    vals = [t.to(cuda()).reshape(S, L, C) for t in tok] + [p.to(cuda()) for p in par]
    dy = randn((S, L, C), g).to(dtype).to(cuda())

    def train():
        v = [t.detach().requires_grad_() for t in vals]
        y = gated_lru_scan(v[0], v[1], v[2], v[4], z=v[3], r_bias=v[5], i_bias=v[6])
        return (y.detach(),) + torch.autograd.grad(y, v, dy)

    want = train()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(train(), want))
    x, r, i, z, rate, rb, ib = vals
    fresh = torch.ones(S, dtype=torch.bool, device=cuda())
    y = gated_lru_scan(x, r, i, rate, z=z, r_bias=rb, i_bias=ib, state=torch.randn(S, C, device=cuda()), fresh=fresh)
    assert torch.equal(y, want[0])
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        train()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = train()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
