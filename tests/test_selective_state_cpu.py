"""Selective state operators on the CPU: the oracle's gradients against autograd and against
differences of its own outputs, refusals that run before any device access, and the mixer's
parameters."""
from __future__ import annotations

import ctypes

import pytest
import torch

from oracle import selective_state as oss
from semambaxlinoss_b200 import _lib
from tests.parity import gen, randn


def _problem(seed, rows=11, ch=6, N=3, G=2, K=3):
    g = gen(seed)
    return {"x": randn((rows, ch), g), "dt": randn((rows, ch), g), "A": -torch.exp(randn((ch, N), g)),
            "B": randn((rows, G, N), g), "C": randn((rows, G, N), g), "D": randn((ch,), g), "z": randn((rows, ch), g),
            "dt_bias": randn((ch,), g), "dy": randn((rows, ch), g), "w": randn((ch, K), g), "b": randn((ch,), g)}


CU = [0, 4, 4, 5, 10]  # a sequence of no rows, one of one, an unused last row


def test_oracle_scan_gradients():
    t = _problem(0)
    names = ("x", "dt", "A", "B", "C", "D", "z", "dt_bias")
    leaves = {k: t[k].clone().requires_grad_() for k in names}
    y = torch.stack([r for r in oss.scan(leaves["x"], leaves["dt"], leaves["A"], leaves["B"], leaves["C"], CU,
                                         leaves["D"], leaves["z"], leaves["dt_bias"])["y"]])
    grads = dict(zip(names, torch.autograd.grad((y * t["dy"]).sum(), [leaves[k] for k in names])))
    args = [t[k] for k in ("x", "dt", "A", "B", "C")]
    out = oss.scan(*args, CU, t["D"], t["z"], t["dt_bias"], dy=t["dy"])
    for k in names:
        torch.testing.assert_close(out["d" + k], grads[k], rtol=1e-11, atol=1e-12)
    # Against differences, one direction for all operands together.
    g, eps = gen(1), 1e-6
    move = {k: randn(t[k].shape, g) for k in names}

    def value(sign):
        v = {k: t[k] + sign * eps * move[k] for k in names}
        return (oss.scan(v["x"], v["dt"], v["A"], v["B"], v["C"], CU, v["D"], v["z"], v["dt_bias"])["y"] * t["dy"]).sum()

    slope = (value(1) - value(-1)) / (2 * eps)
    torch.testing.assert_close(sum((out["d" + k] * move[k]).sum() for k in names), slope, rtol=1e-7, atol=1e-8)


def test_oracle_conv_gradients():
    t = _problem(2)
    leaves = [t[k].clone().requires_grad_() for k in ("x", "w", "b")]
    y = torch.stack([r for r in oss.conv(*leaves, CU)["y"]])
    grads = torch.autograd.grad((y * t["dy"]).sum(), leaves)
    out = oss.conv(t["x"], t["w"], t["b"], CU, dy=t["dy"])
    for k, g in zip(("dx", "dw", "db"), grads):
        torch.testing.assert_close(out[k], g, rtol=1e-11, atol=1e-12)
    # A sequence in two calls equals the sequence in one.
    whole = oss.conv(t["x"], t["w"], t["b"], [0, 11])
    first = oss.conv(t["x"][:4], t["w"], t["b"], [0, 4])
    second = oss.conv(t["x"][4:], t["w"], t["b"], [0, 7], windows=first["windows"])
    torch.testing.assert_close(torch.cat([first["y"], second["y"]]), whole["y"])


def test_cpu_tensors_are_refused():
    from semambaxlinoss_b200.selective_state import (selective_state_scan, selective_state_step, short_conv,
                                                     short_conv_step)

    x, w = torch.randn(2, 5, 8), torch.randn(8, 4)
    with pytest.raises(RuntimeError):
        short_conv(x, w)
    with pytest.raises(RuntimeError):
        short_conv_step(x[0], torch.zeros(5, 3, 8), w)
    BC = torch.randn(2, 5, 4)
    with pytest.raises(RuntimeError):
        selective_state_scan(x, x, torch.randn(8, 4), BC, BC)
    with pytest.raises(RuntimeError):
        selective_state_step(x[0], x[0], torch.randn(8, 4), BC[0], BC[0], torch.zeros(5, 8, 4))


def _status(entry, cls, base, **fields):
    a = _lib.new_args(cls)
    for k, v in {**base, **fields}.items():
        setattr(a, k, v)
    return getattr(_lib.load(), entry)(ctypes.byref(a), None)


def test_conv_status_codes():
    cls, base = _lib.SemxShortConvArgs, dict(K=4, S=2, rows=10, L=5, C=8, ldx=8)
    fwd = lambda **f: _status("semx_short_conv_fwd", cls, base, **f)  # noqa: E731
    bwd = lambda **f: _status("semx_short_conv_bwd", cls, base, **f)  # noqa: E731
    assert fwd(struct_size=4) == _lib.SEMX_ERR_ABI
    assert fwd() == _lib.SEMX_ERR_NULL
    for bad in (dict(K=0), dict(K=9)):
        assert fwd(**bad) == _lib.SEMX_ERR_UNSUPPORTED
    ptr = dict(x=256, w=256, y=256)
    for bad in (dict(C=0), dict(ldx=7), dict(rows=11), dict(S=-1), dict(rows=2 ** 31, S=2 ** 31, L=1), dict(n_slots=-1),
                dict(state=256, n_slots=1), dict(ldx=2 ** 31)):
        assert fwd(**ptr, **bad) == _lib.SEMX_ERR_SHAPE, bad
    for bad in (dict(state=256), dict(n_slots=2), dict(slots=256), dict(fresh=256)):
        assert fwd(**ptr, **bad) == _lib.SEMX_ERR_NULL, bad
    for bad in (dict(x=257), dict(y=258), dict(w=258), dict(slots=257, state=256, n_slots=2)):
        assert fwd(**{**ptr, **bad}) == _lib.SEMX_ERR_ALIGN, bad
    assert fwd(**{**ptr, "x": 257}, bf16=1) == _lib.SEMX_ERR_ALIGN
    assert bwd(**ptr, dy=256) == _lib.SEMX_ERR_NULL
    assert bwd(**ptr, dy=256, dx=256, dw=256) == _lib.SEMX_ERR_WORKSPACE
    assert bwd(**ptr, dy=256, dx=256, state=256, n_slots=2) == _lib.SEMX_ERR_UNSUPPORTED


def test_scan_status_codes():
    cls = _lib.SemxStateScanArgs
    base = dict(S=2, rows=10, L=5, C=8, N=4, G=2, ldx=8, lddt=8, ldb=8, ldc=8)
    ptr = dict(x=256, dt=256, A=256, B=256, Cm=256, y=256)
    fwd = lambda **f: _status("semx_state_scan_fwd", cls, base, **f)  # noqa: E731
    assert fwd(struct_size=4) == _lib.SEMX_ERR_ABI
    assert fwd() == _lib.SEMX_ERR_NULL
    for bad in (dict(N=0), dict(N=129)):
        assert fwd(**ptr, **bad) == _lib.SEMX_ERR_UNSUPPORTED
    for bad in (dict(C=0), dict(G=3), dict(G=0), dict(ldx=7), dict(ldb=7), dict(z=256, ldz=7), dict(rows=9),
                dict(state=256, n_slots=1)):
        assert fwd(**ptr, **bad) == _lib.SEMX_ERR_SHAPE, bad
    for bad in (dict(x=258), dict(dt=257, dt_bf16=1), dict(A=258), dict(state=258, n_slots=2)):
        assert fwd(**{**ptr, **bad}) == _lib.SEMX_ERR_ALIGN, bad
    assert _status("semx_state_scan_bwd", cls, base, **ptr, dy=256) == _lib.SEMX_ERR_NULL
    back = dict(ptr, dy=256, dx=256, ddt=256, dB=256, dC=256, ckpt=256)
    assert _status("semx_state_scan_bwd", cls, base, **back) == _lib.SEMX_ERR_WORKSPACE
    assert _status("semx_state_scan_bwd", cls, base, **back, z=256, ldz=8) == _lib.SEMX_ERR_NULL
    assert _status("semx_state_scan_bwd", cls, base, **back, state=256, n_slots=2) == _lib.SEMX_ERR_UNSUPPORTED
    step = dict(base, rows=2, L=1)
    assert _status("semx_state_step", cls, base, **ptr, state=256, n_slots=2) == _lib.SEMX_ERR_SHAPE
    assert _status("semx_state_step", cls, step, **ptr) == _lib.SEMX_ERR_NULL


def test_sizes():
    lib = _lib.load()
    a = _lib.new_args(_lib.SemxStateScanArgs)
    a.S, a.rows, a.L, a.C, a.N, a.G = 3, 30, 10, 8, 4, 1
    a.ldx = a.lddt = 8
    a.ldb = a.ldc = 4
    assert lib.semx_state_scan_ckpt_bytes(ctypes.byref(a)) == 3 * 2 * 8 * 4 * 4  # every 8th step's state
    a.cu_seqlens, a.L = 256, 0
    assert lib.semx_state_scan_ckpt_bytes(ctypes.byref(a)) == (30 // 8 + 3) * 8 * 4 * 4
    assert lib.semx_state_scan_workspace_bytes(ctypes.byref(a), 1) > 0
    a.C = 0
    assert lib.semx_state_scan_workspace_bytes(ctypes.byref(a), 1) == 0


def test_piece_numbers_hold_every_sequence():
    """The numbering of pieces that the kernels use, checked on the CPU: pieces of Q rows of a
    packed batch start at cu[s] // Q + s, never overlap and fit rows // Q + S numbers."""
    g = torch.Generator().manual_seed(0)
    for case in range(200):
        S, Q = int(torch.randint(1, 9, (1,), generator=g)), int(2 ** torch.randint(0, 7, (1,), generator=g))
        lens = torch.randint(0, 40, (S,), generator=g) * (torch.rand(S, generator=g) < 0.8)
        cu = [0] + torch.cumsum(lens, 0).tolist()
        T = cu[-1] + case % 3
        used = set()
        for s in range(S):
            for k in range(-(-int(lens[s]) // Q)):
                j = cu[s] // Q + s + k
                assert j not in used and j < T // Q + S
                used.add(j)
                # The search takes the last sequence whose first piece is not behind j.
                assert max(i for i in range(S) if cu[i] // Q + i <= j) == s


def test_mixer_parameters_and_factory():
    from semambaxlinoss_b200.selective_state import SelectiveStateMixer

    m = SelectiveStateMixer(32, d_state=8, d_conv=3, expand=2, n_groups=2)
    assert list(m.state_dict()) == ["A_log", "D", "in_proj.weight", "conv1d.weight", "conv1d.bias", "x_proj.weight",
                                    "dt_proj.weight", "dt_proj.bias", "out_proj.weight"]
    assert m.conv1d.weight.shape == (64, 1, 3) and m.x_proj.weight.shape == (2 + 2 * 2 * 8, 64)
    dt = torch.nn.functional.softplus(m.dt_proj.bias)
    assert (dt >= 1e-3 - 1e-6).all() and (dt <= 0.1 + 1e-6).all()
    assert m.A_log._no_weight_decay and m.D._no_weight_decay and m.dt_proj.bias._no_reinit
    c = m.allocate_cache(5)
    assert c.window.shape == (5, 2, 64) and c.state.shape == (5, 64, 8) and c.state.dtype == torch.float32
    with pytest.raises(ValueError):
        SelectiveStateMixer(33, n_groups=4, expand=1)
    with pytest.raises(RuntimeError):
        m(torch.randn(2, 5, 32))
