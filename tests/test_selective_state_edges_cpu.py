"""What the selective state operators' entry points answer before any device access, on the CPU."""
from __future__ import annotations

import pytest

from semambaxlinoss_b200 import _lib
from tests.test_selective_state_cpu import _status


@pytest.mark.parametrize("S,cu", [(3, 0), (0, 0), (3, 256), (0, 256)])
def test_an_empty_forward_launches_nothing(S, cu):
    """No rows and no pool: there is no output whose address names the GPU, and nothing to write. The
    call must not run a kernel on whichever GPU is current (here there is none, so a launch
    would come back as an error)."""
    before = _lib.launch_count()
    conv = dict(K=4, S=S, rows=0, L=0, C=8, ldx=8, w=256, cu_seqlens=cu)
    scan = dict(S=S, rows=0, L=0, C=8, N=4, G=2, ldx=8, lddt=8, ldb=8, ldc=8, A=256, cu_seqlens=cu)
    assert _status("semx_short_conv_fwd", _lib.SemxShortConvArgs, conv) == _lib.SEMX_OK
    assert _status("semx_short_conv_fwd", _lib.SemxShortConvArgs, conv, K=1, state=256, n_slots=3) == _lib.SEMX_OK
    assert _status("semx_short_conv_bwd", _lib.SemxShortConvArgs, conv) == _lib.SEMX_OK
    assert _status("semx_state_scan_fwd", _lib.SemxStateScanArgs, scan) == _lib.SEMX_OK
    assert _status("semx_state_scan_bwd", _lib.SemxStateScanArgs, scan, workspace=256) == _lib.SEMX_OK
    assert _lib.launch_count() == before
