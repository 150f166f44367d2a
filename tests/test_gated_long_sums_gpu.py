"""Weight gradients of the bf16 gated projection over very many rows whose terms have one sign: their sums do not
stay in the tensor cores, which cut where an addition rounds."""
from __future__ import annotations

import pytest
import torch

from tests.parity import cuda

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,D,H", [(131072, 1024, 1408), (70001, 200, 1800), (129684, 64, 256)])
def test_bf16_weight_gradient_of_many_rows(rows, D, H):
    """Every value is within half a step of its own binade, and 1e-4: the tensor cores take some hundred additions at
    a time, each at most 4 eps (the sum's and the aligned terms' cut, 2 eps each) of a partial sum that is half of its
    run on average, so 3e-5 for 256 of them; du and dg are rounded, 2^-8 over the root of the rows: 1.5e-5; fp32
    additions of the runs 1e-5. (One sum over 131072 rows is 7e-4 too small.)"""
    from semambaxlinoss_b200.gated_mlp import gated_linear

    g = torch.Generator(device="cuda").manual_seed(rows)

    def rand(*shape):
        return torch.rand(*shape, generator=g, device=cuda())

    x = ((rand(rows, D) + 0.5) * 2 ** rand(D)).bfloat16()  # columns of many sizes, so that results lie anywhere in a step
    w = ((rand(2 * H, D) + 0.5) / D).bfloat16().requires_grad_()
    dh = ((rand(rows, H) + 0.5) * 2 ** rand(H)).bfloat16()
    (dw,) = torch.autograd.grad(gated_linear(x, w), w, dh)
    n = 24
    want = torch.zeros(2 * n, D, dtype=torch.float64, device=cuda())
    for r in range(0, rows, 16384):
        xs, d = x[r:r + 16384].double(), dh[r:r + 16384, :n].double()
        u, v = xs @ w.detach()[:n].double().t(), xs @ w.detach()[H:H + n].double().t()
        s = torch.sigmoid(v)
        want += torch.cat([d * v * s, d * u * s * (1 + v * (1 - s))], 1).t() @ xs
    got = torch.cat([dw[:n], dw[H:H + n]]).double()
    half = torch.exp2(torch.floor(torch.log2(want)) - 8)
    over = (got - want).abs() - half - 1e-4 * want
    assert bool((over <= 0).all()), (over / want).max().item()
