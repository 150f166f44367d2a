"""Selective state operators on the GPU at the ends of what a call may ask for, against the
float64 oracle. Tolerances as derived in test_selective_state_gpu.py."""
from __future__ import annotations

import pytest
import torch

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
