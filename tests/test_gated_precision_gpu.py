"""The fp32 gated projection keeps fp32's precision: root mean square errors against float64, with bounds that
sums without the small parts, or left in the tensor cores, do not meet (test_gated_precision_cpu.py)."""
from __future__ import annotations

import pytest
import torch

from tests import gated_precision as gp
from tests.parity import cuda

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("case", gp.CASES)
def test_fp32_precision(case):
    from semambaxlinoss_b200.gated_mlp import gated_linear

    signs, rows, D, H = case
    x, w, dh = gp.inputs(*case)
    want = gp.exact(x, w, dh)
    ins = [t.to(cuda()).requires_grad_() for t in (x, w)]
    h = gated_linear(*ins)
    dx, dw = torch.autograd.grad(h, ins, dh.to(cuda()))
    for name, got in (("h", h.detach()), ("dx", dx), ("dw", dw)):
        off = gp.off(got, want[name])
        assert off <= gp.allowed(name, rows, D, H), (name, off, gp.allowed(name, rows, D, H))


@pytest.mark.parametrize("rows", [1, 3, 8, 16])
def test_fp32_precision_of_few_rows(rows):
    """Few rows are summed in fp32 throughout: D / 64 additions a lane in two halves, and 6 across the lanes."""
    from semambaxlinoss_b200.gated_mlp import gated_linear

    for signs, D, H in (("random", 1000, 40), ("same", 6000, 24)):
        x, w, dh = gp.inputs(signs, rows, D, H)
        h = gated_linear(x.to(cuda()), w.to(cuda()))
        assert gp.off(h, gp.exact(x, w, dh)["h"]) <= gp.allowed("h", rows, D, H)
