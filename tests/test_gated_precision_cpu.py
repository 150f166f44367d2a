"""The bounds of the fp32 gated projection's precision hold for its sums as they are taken, and fail where parts'
products are left out or long sums stay in the tensor cores: a model of both on the CPU."""
from __future__ import annotations

import pytest

from tests import gated_precision as gp

# The result whose product is long, of the cases with one sign.
LONG = {6000: "h", 3500: "dx", 24000: "dw"}


@pytest.mark.parametrize("case", gp.CASES)
def test_bounds(case):
    signs, rows, D, H = case
    ins = gp.inputs(*case)
    want = gp.exact(*ins)

    def over(**kw):
        return {n for n, v in gp.model(*ins, **kw).items() if gp.off(v, want[n]) > gp.allowed(n, rows, D, H)}

    assert over() == set()
    assert over(products=1) == {"h", "dx", "dw"}
    if signs == "random":
        assert over(products=3) == over(products=4) == {"h", "dx", "dw"}
    else:
        assert LONG[max(rows, D, H)] in over(drain=0)
