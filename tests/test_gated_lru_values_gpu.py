"""Gated recurrence on the GPU at values where a formula in 32 bits can go wrong although the result is
an ordinary number: gates shut by the type's lowest value, rates whose speed is below the normal
numbers, and gates that are no number. Tolerances as in test_gated_lru_gpu.py."""
from __future__ import annotations

import pytest
import torch

from oracle import gated_lru as ogl
from tests.parity import cuda, gen, randn
from tests.test_gated_lru_gpu import EPS, HALF

pytestmark = pytest.mark.gpu
NAMES = ("y", "dx", "dr", "di", "dz")


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_shut_gates_pass_nothing_back(packed, dtype):
    """Output gates z, input gates i (beside large inputs) and decay gates r at and near the lowest value:
    a shut gate's gradient is 0, whatever it shuts. A sigmoid below 2^-126 counts as 0: times 1 + |z|, at
    most 104 where fp32 has such a sigmoid at all, that is 2^-119 of what it multiplies (here up to 2^7)."""
    from semambaxlinoss_b200.gated_lru import gated_lru_scan

    low = torch.finfo(dtype).min
    shut = [low, low / 4, -1e37, -1e30, -1e10, -1e4, -200.0, -90.0, -88.0, -87.0, -60.0, -20.0, 0.0, 20.0, 200.0, 1e30]
    g = gen(51)
    L, n = 70, len(shut)
    C = 3 * n
    x, r, i, z, dy = (randn((L, C), g).to(dtype).double() for _ in range(5))
    gate = torch.tensor(shut, dtype=torch.float64).to(dtype).double()
    z[:, :n] = gate
    i[:, n:2 * n] = gate
    r[:, 2 * n:] = gate
    x[:, n:n + 4] = torch.finfo(dtype).max / 2  # behind input gates that are shut
    rate = torch.full((C,), -3.0, dtype=torch.float64)
    want = ogl.scan(x, r, i, rate, [0, L], z, dy=dy)
    size = ogl.scan(x, r, i, rate, [0, L], z, dy=dy, absolute=True)
    cu = torch.tensor([0, L], dtype=torch.int32, device=cuda()) if packed else None
    d = [t.to(dtype).to(cuda()) for t in (x, r, i, z)]
    d = [(t if packed else t[None]).requires_grad_() for t in d]
    rd = rate.float().to(cuda()).requires_grad_()
    y = gated_lru_scan(d[0], d[1], d[2], rd, z=d[3], cu_seqlens=cu)
    grads = torch.autograd.grad(y, d + [rd], dy.to(dtype).to(cuda()).reshape(y.shape))
    for name, got in zip(NAMES + ("drate",), (y,) + grads):
        got = got.detach().double().cpu().reshape(want[name].shape)
        half = HALF[torch.float32 if name == "drate" else dtype]
        tol = (24 * L + 256 + L) * EPS * size[name] + half * want[name].abs() + 2.0 ** -112
        assert torch.isfinite(got).all(), name
        over = (got - want[name]).abs() - tol
        assert bool((over <= 0).all()), (name, over.max().item(), int(over.argmax()) % C)


@pytest.mark.parametrize("packed", [False, True])
def test_speeds_below_the_normal_numbers(packed):
    """rate_scale softplus(rate) among fp32's subnormal numbers, or 0: the decay is 1 and the gain its least
    value, 1e-3, for whole sequences, their gradients and single tokens. Sums over three steps in fp32, each of
    at most 8 roundings: 24 eps of terms that do not cancel here, 2e-6 allowed."""
    from semambaxlinoss_b200.gated_lru import gated_lru_scan, gated_lru_step

    rate = torch.linspace(-92, -82, 41, dtype=torch.float64).repeat(2)[:72]
    C, L, scale = rate.numel(), 3, 0.1
    g = gen(52)
    x, dy = randn((L, C), g).abs().float().double(), randn((L, C), g).abs().float().double()
    r, i = torch.full((L, C), 3.0, dtype=torch.float64), torch.full((L, C), 0.5, dtype=torch.float64)
    want = ogl.scan(x, r, i, rate.float().double(), [0, L], scale=scale, dy=dy)
    cu = torch.tensor([0, L], dtype=torch.int32, device=cuda()) if packed else None
    d = [t.float().to(cuda()) for t in (x, r, i)]
    d = [(t if packed else t[None]).requires_grad_() for t in d]
    rd = rate.float().to(cuda()).requires_grad_()
    y = gated_lru_scan(d[0], d[1], d[2], rd, rate_scale=scale, cu_seqlens=cu)
    grads = torch.autograd.grad(y, d + [rd], dy.float().to(cuda()).reshape(y.shape))
    state = torch.zeros(1, C, device=cuda())
    toks = torch.cat([gated_lru_step(*(t.detach().reshape(L, C)[k:k + 1] for t in d), rd.detach(), state, rate_scale=scale)
                      for k in range(L)])
    for name, got in zip(("y", "dx", "dr", "di", "drate", "y"), (y,) + grads + (toks,)):
        got = got.detach().double().cpu().reshape(want[name].shape)
        assert torch.isfinite(got).all(), name
        assert torch.allclose(got, want[name], rtol=2e-6, atol=1e-30), (name, (got - want[name]).abs().max())


@pytest.mark.parametrize("gate", ["r", "i"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gates_that_are_no_number(gate, dtype):
    """A NaN among the gates of one step: NaN where the formulas have it, and the other channels as without it."""
    from semambaxlinoss_b200.gated_lru import gated_lru_scan

    g = gen(53)
    L, C, at, ch = 150, 40, 70, 9
    tok = {n: randn((L, C), g).to(dtype) for n in ("x", "r", "i", "z")}
    rate, dy = torch.full((C,), -5.0), randn((L, C), g).to(dtype)

    def run(tok):
        d = [tok[n].to(cuda())[None].requires_grad_() for n in ("x", "r", "i", "z")]
        rd = rate.to(cuda()).requires_grad_()
        y = gated_lru_scan(d[0], d[1], d[2], rd, z=d[3])
        return [t.detach().cpu().reshape(-1, C) for t in (y,) + torch.autograd.grad(y, d + [rd], dy.to(cuda())[None])]

    clean = run(tok)
    tok[gate][at, ch] = float("nan")
    t64 = {n: t.double() for n, t in tok.items()}
    want = ogl.scan(t64["x"], t64["r"], t64["i"], rate.double(), [0, L], t64["z"], dy=dy.double())
    others = torch.arange(C) != ch
    for name, got, was in zip(NAMES + ("drate",), run(tok), clean):
        assert torch.equal(torch.isnan(got), torch.isnan(want[name].reshape(got.shape))), name
        assert torch.equal(got[:, others], was[:, others]), name
