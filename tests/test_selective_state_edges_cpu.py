"""What the selective state operators' entry points answer before any device access, on the CPU."""
from __future__ import annotations

import pytest
import torch

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


def test_tangents_are_refused_inside_a_dual_level_only():
    from torch.autograd import forward_ad

    x, w = torch.randn(3), torch.randn(3)
    _lib.refuse_tangents("op", x, None, w)
    with forward_ad.dual_level():
        _lib.refuse_tangents("op", x, None, w)
        d = forward_ad.make_dual(x, torch.ones(3))
        for operands in ((d,), (w, None, d), (w, d[1:])):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError, match="^op: "):
                    _lib.refuse_tangents("op", *operands)
    _lib.refuse_tangents("op", d)  # outside of its level a dual tensor is a plain one


def test_the_mixer_refuses_slots_without_a_cache():
    """As the operators below it do without a state; neither is dropped."""
    from semambaxlinoss_b200.selective_state import SelectiveStateMixer

    mixer, x = SelectiveStateMixer(8), torch.randn(2, 5, 8)
    for bad in (dict(slots=torch.zeros(2, dtype=torch.int32)), dict(fresh=torch.ones(2, dtype=torch.bool))):
        with pytest.raises(ValueError, match="without a cache"):
            mixer(x, **bad)


@pytest.mark.parametrize("default", [torch.bfloat16, torch.float64])
def test_the_state_is_fp32_under_any_default_type(default):
    """A model built under torch.set_default_dtype gets the cache that the scan takes."""
    from semambaxlinoss_b200.selective_state import SelectiveStateMixer

    before = torch.get_default_dtype()
    torch.set_default_dtype(default)
    try:
        mixer = SelectiveStateMixer(8)
        cache = mixer.allocate_cache(3)
    finally:
        torch.set_default_dtype(before)
    assert mixer.in_proj.weight.dtype == cache.window.dtype == default
    assert cache.state.dtype == torch.float32 and not cache.state.any()


def test_the_factory_names_the_selective_state_mixer():
    from semambaxlinoss_b200.mamba_block import create_block

    cfg = {"d_state": 4, "d_conv": 4, "expand": 2}
    for name in ("mamba", "s4d"):
        with pytest.raises(NotImplementedError, match="selective state mixer") as e:
            create_block(8, dict(cfg, ssm=name))
        assert ("'selective_state'" in str(e.value)) == (name == "mamba")
    with pytest.raises(ValueError, match="'selective_state'"):
        create_block(8, dict(cfg, ssm="unknown"))
