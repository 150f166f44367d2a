"""The gated projection's workspace: what a size query covers, and that a call which needs more than it is given
is refused on the host, before anything runs on a GPU."""
from __future__ import annotations

import ctypes

import pytest

from semambaxlinoss_b200 import _lib

SIZES = [(rows, D, H, bf16) for rows in (1, 5, 12, 16, 17, 300, 5000) for D, H in ((64, 40), (72, 33), (1000, 264), (71, 9))
         for bf16 in (0, 1)]


def _args(rows, D, H, bf16, backward, x=4096, w=4096, grads="dx dw db", **kw):
    a = _lib.new_args(_lib.SemxGatedLinearArgs)
    a.rows, a.D, a.H, a.ldx, a.bf16 = rows, D, H, D, bf16
    a.x, a.w, a.h = x, w, 4096
    if backward:
        a.h, a.dh, a.saved = None, 4096, 4096
        for n in grads.split():
            setattr(a, n, 4096)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _bytes(a, backward):
    return _lib.load().semx_gated_linear_workspace_bytes(ctypes.byref(a), backward)


def _call(a, backward):
    return getattr(_lib.load(), "semx_gated_linear_bwd" if backward else "semx_gated_linear_fwd")(ctypes.byref(a), None)


@pytest.mark.parametrize("backward", [0, 1])
def test_a_query_without_addresses_covers_every_address(backward):
    for size in SIZES:
        step = 2 if size[3] else 4
        most = _bytes(_args(*size, backward, x=None, w=None), backward)
        for x in (4096, 4096 + step):
            for w in (4096, 4096 + step):
                need = _bytes(_args(*size, backward, x=x, w=w), backward)
                assert need <= most, (size, x, w)
                assert _bytes(_args(*size, backward, x=None, w=w), backward) >= need
                assert _bytes(_args(*size, backward, x=x, w=None), backward) >= need


@pytest.mark.parametrize("backward", [0, 1])
def test_too_small_a_workspace_is_refused(backward):
    """Bases off 16 bytes with the bytes of a query on 16, more gradients than the query had, one byte less, none."""
    seen = 0
    for size in SIZES:
        step = 2 if size[3] else 4
        given = [_bytes(_args(*size, backward), backward)]
        if backward:
            given += [_bytes(_args(*size, backward, grads=g), backward) for g in ("dx", "dw", "db")]
        for off_x, off_w in ((0, 0), (step, 0), (0, step), (step, step)):
            kw = dict(x=4096 + off_x, w=4096 + off_w, workspace=4096)
            need = _bytes(_args(*size, backward, **kw), backward)
            for n in given + [need - 1, 0, -1]:
                if n >= need or need == 0:
                    continue
                seen += 1
                assert _call(_args(*size, backward, **kw, workspace_bytes=n), backward) == _lib.SEMX_ERR_WORKSPACE, (size, n)
            if need:
                kw["workspace"] = None
                assert _call(_args(*size, backward, **kw, workspace_bytes=need), backward) == _lib.SEMX_ERR_WORKSPACE
    assert seen > 100


def test_what_a_call_refuses_has_no_size():
    for kw in (dict(D=0), dict(H=0), dict(rows=-1), dict(D=1 << 40), dict(H=1 << 40), dict(rows=1 << 40), dict(ldx=3)):
        a = _args(300, 64, 40, 1, 0)
        for k, v in kw.items():
            setattr(a, k, v)
        assert _bytes(a, 0) == 0, kw


def test_no_gradients_wanted_needs_nothing():
    assert _call(_args(300, 64, 40, 1, 1, grads=""), 1) == _lib.SEMX_OK
