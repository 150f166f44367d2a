"""Gated recurrence and gated projection in batches that are partly padding, under autocast and from autograd's
own thread, against the float64 oracle or the plain call. Tolerances as in test_gated_lru_gpu.py."""
from __future__ import annotations

import pytest
import torch

from tests.parity import assert_close, cuda, gen, randn
from tests.test_gated_lru_gpu import _near, _operands, _oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("C", [24, 7, 130])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_of_no_sequence_hold_anything(C, dtype):
    """NaN and infinities in front of the first sequence and behind the last one, in every operand and in dy: zeros
    come out there, and nothing of them in the sequences or the sums over rows."""
    from semambaxlinoss_b200.gated_lru import gated_lru_scan

    cu, rows = [37, 40, 40, 240, 241, 306], 350
    g = gen(C)
    tok, par = _operands(rows, C, dtype, g)
    dy = randn((rows, C), g).to(dtype)
    want, size = _oracle(tok, par, cu, dy=dy.double())
    out = [slice(0, cu[0]), slice(cu[-1], rows)]
    for k, t in enumerate(tok + [dy]):
        for s in out:
            t[s] = float("nan") if k % 2 else float("inf")
    dev = [t.to(cuda()).requires_grad_() for t in tok]
    pd = [p.to(cuda()).requires_grad_() for p in par]
    y = gated_lru_scan(dev[0], dev[1], dev[2], pd[0], z=dev[3], r_bias=pd[1], i_bias=pd[2],
                       cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=cuda()))
    grads = torch.autograd.grad(y, dev + pd, dy.to(cuda()))
    _near(y, want["y"], size["y"], 10 * 200 + 96, dtype, "y")
    for name, got in zip(("dx", "dr", "di", "dz", "drate", "dr_bias", "di_bias"), grads):
        whole = got.dim() == 1
        _near(got, want[name], size[name], 24 * 200 + 256 + (rows if whole else 0), torch.float32 if whole else dtype, name)
        if not whole:
            assert not any(got[s].any() for s in out), name
    assert not any(y[s].any() for s in out)


@pytest.mark.parametrize("C", [40, 9])
@pytest.mark.parametrize("S,L", [(3, 150), (600, 70)])
def test_a_sequence_that_is_no_number_stays_alone(S, L, C):
    """NaN in one sequence of a batch: the others' outputs, states and row gradients keep their bits, linked and
    walked."""
    from semambaxlinoss_b200.gated_lru import gated_lru_scan

    g = gen(S + C)
    tok, par = _operands(S * L, C, torch.float32, g)
    vals = [t.to(cuda()).reshape(S, L, C) for t in tok]
    rate, dy = par[0].to(cuda()), randn((S, L, C), g).float().to(cuda())
    others = [s for s in range(S) if s != 1]

    def run(vals):
        v = [t.clone().requires_grad_() for t in vals]
        y = gated_lru_scan(v[0], v[1], v[2], rate, z=v[3])
        grads = torch.autograd.grad(y, v, dy)
        state = torch.zeros(S, C, device=cuda())
        p = gated_lru_scan(*vals[:3], rate, z=vals[3], state=state)
        return [t.detach()[others] for t in (y, *grads, p, state)]

    clean = run(vals)
    for k in range(4):
        bad = [t.clone() for t in vals]
        bad[k][1, L // 2] = float("nan")
        assert all(torch.equal(a, b) for a, b in zip(run(bad), clean)), k


def test_blocks_under_autocast():
    """fp32 parameters under bf16 autocast: near the fp32 pass (ten roundings of 2^-8 on the way), gradients in fp32."""
    from semambaxlinoss_b200.mamba_block import MambaBlock

    torch.manual_seed(2)
    cfg = {"ssm": "gated_lru", "d_state": 4, "d_conv": 4, "expand": 2, "mlp": {}}
    m = MambaBlock(64, cfg).to(cuda())
    x = randn((2, 90, 64), gen(3)).float().to(cuda())
    dy = randn((2, 90, 128), gen(4)).float().to(cuda())
    want = m(x)
    wg = torch.autograd.grad(want, list(m.parameters()), dy)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        got = m(x)
    gg = torch.autograd.grad(got, list(m.parameters()), dy.to(got.dtype))
    assert_close(got.float(), want, 4e-2)
    for (name, p), a, b in zip(m.named_parameters(), gg, wg):
        assert a.dtype == p.dtype
        assert float((a - b).norm() / b.norm()) <= 4e-2, name
    cache = m.forward_blocks[0].mixer.allocate_cache(2, dtype=torch.bfloat16)
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        whole = sum(m.forward_blocks[0](x))
        fresh = torch.ones(2, dtype=torch.bool, device=cuda())
        head = sum(m.forward_blocks[0](x[:, :89], cache=cache, fresh=fresh))
        last = sum(m.forward_blocks[0](x[:, 89:], cache=cache))
    assert_close(torch.cat([head, last], 1).float(), whole.float(), 4e-2)


def test_backward_twice_and_in_place_changes():
    """A kept graph gives the same gradients again; operands changed in place since are noticed."""
    from semambaxlinoss_b200.gated_lru import gated_lru_scan
    from semambaxlinoss_b200.gated_mlp import gated_linear

    g = gen(5)
    x, r, i, z = (randn((2, 70, 24), g).float().to(cuda()).requires_grad_() for _ in range(4))
    w = randn((40, 24), g).float().to(cuda()).requires_grad_()
    rate = torch.full((24,), -4.0, device=cuda(), requires_grad=True)
    for call, ins in ((lambda: gated_lru_scan(x, r, i, rate, z=z), (x, r, i, z, rate)), (lambda: gated_linear(x, w), (x, w))):
        y = call()
        dy = torch.ones_like(y)
        first = torch.autograd.grad(y, ins, dy, retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, ins, dy), first))
        y = call()
        with torch.no_grad():
            ins[1].add_(1.0)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            torch.autograd.grad(y, ins, dy)
