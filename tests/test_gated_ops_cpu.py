"""Gated recurrence and gated projection without a GPU: refusals of the operators and the library,
size queries, factory, initial values, oracles against autograd."""
from __future__ import annotations

import ctypes

import pytest
import torch

from oracle import gated_lru as ogl
from oracle import gated_mlp as ogm
from semambaxlinoss_b200 import _lib
from tests.parity import gen, randn


def test_cpu_tensors_are_refused():
    from semambaxlinoss_b200.gated_lru import gated_lru_scan, gated_lru_step
    from semambaxlinoss_b200.gated_mlp import gated_linear

    x = torch.zeros(2, 3, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        gated_lru_scan(x, x, x, torch.zeros(8))
    with pytest.raises(RuntimeError, match="CUDA"):
        gated_lru_step(x[:, 0], x[:, 0], x[:, 0], torch.zeros(8), torch.zeros(2, 8))
    with pytest.raises(RuntimeError, match="CUDA"):
        gated_linear(x, torch.zeros(8, 8))


def _lru_args():
    a = _lib.new_args(_lib.SemxGatedLruArgs)
    a.S, a.rows, a.L, a.C, a.rate_scale = 2, 200, 100, 12, 8.0
    a.ldx = a.ldr = a.ldi = a.ldz = 12
    for n in ("x", "r", "i", "rate", "y"):
        setattr(a, n, 4096)
    return a


def test_recurrence_arguments_are_checked_on_the_host():
    lib = _lib.load()

    def status(fn="semx_gated_lru_fwd", **kw):
        a = _lru_args()
        for k, v in kw.items():
            setattr(a, k, v)
        return getattr(lib, fn)(ctypes.byref(a), None)

    assert status(struct_size=3) == _lib.SEMX_ERR_ABI
    assert status(C=0) == _lib.SEMX_ERR_SHAPE
    assert status(ldx=11) == _lib.SEMX_ERR_SHAPE
    assert status(z=4096, ldz=5) == _lib.SEMX_ERR_SHAPE
    assert status(rows=199) == _lib.SEMX_ERR_SHAPE
    assert status(rate_scale=0.0) == _lib.SEMX_ERR_SHAPE
    assert status(rate_scale=float("nan")) == _lib.SEMX_ERR_SHAPE
    assert status(r=None) == _lib.SEMX_ERR_NULL
    assert status(y=None) == _lib.SEMX_ERR_NULL
    assert status(slots=4096) == _lib.SEMX_ERR_NULL
    assert status(state=4096) == _lib.SEMX_ERR_NULL
    assert status(x=4097) == _lib.SEMX_ERR_ALIGN
    assert status("semx_gated_lru_bwd") == _lib.SEMX_ERR_NULL
    assert status("semx_gated_lru_bwd", state=4096, n_slots=2) == _lib.SEMX_ERR_UNSUPPORTED
    assert status("semx_gated_lru_step", L=100) == _lib.SEMX_ERR_SHAPE
    assert status("semx_gated_lru_step", rows=2, L=1) == _lib.SEMX_ERR_NULL
    assert status("semx_gated_lru_step", rows=2, L=1, state=4096, n_slots=2, fresh=4096) == _lib.SEMX_ERR_UNSUPPORTED
    # No rows, no pool: nothing to launch.
    assert status(S=0, rows=0) == _lib.SEMX_OK


def test_recurrence_sizes():
    lib = _lib.load()
    a = _lru_args()
    # A kept state every 32 steps. Linked: a map (16 bytes) and a state (8) per tile of 64 steps (backward
    # 32) and channel, and a ticket per 32 channels.
    assert lib.semx_gated_lru_ckpt_bytes(ctypes.byref(a)) == 2 * 4 * 12 * 4
    assert lib.semx_gated_lru_workspace_bytes(ctypes.byref(a), 0) == 16 + 4 * 12 * 24
    assert lib.semx_gated_lru_workspace_bytes(ctypes.byref(a), 1) == 16 + 8 * 12 * 24 + 8 * 3 * 12 * 4
    a.S, a.rows = 1000, 100000  # sequences enough to walk them
    assert lib.semx_gated_lru_workspace_bytes(ctypes.byref(a), 0) == 0
    assert lib.semx_gated_lru_workspace_bytes(ctypes.byref(a), 1) == 1000 * 3 * 12 * 4
    a.S, a.rows, a.L = 10, 200, 20  # one tile each
    assert lib.semx_gated_lru_workspace_bytes(ctypes.byref(a), 0) == 0


def test_projection_arguments_are_checked_on_the_host():
    lib = _lib.load()

    def status(fn="semx_gated_linear_fwd", **kw):
        a = _lib.new_args(_lib.SemxGatedLinearArgs)
        a.rows, a.D, a.H, a.ldx = 5, 16, 8, 16
        a.x = a.w = a.h = 4096
        for k, v in kw.items():
            setattr(a, k, v)
        return getattr(lib, fn)(ctypes.byref(a), None)

    assert status(struct_size=3) == _lib.SEMX_ERR_ABI
    assert status(D=0) == _lib.SEMX_ERR_SHAPE
    assert status(H=0) == _lib.SEMX_ERR_SHAPE
    assert status(rows=-1) == _lib.SEMX_ERR_SHAPE
    assert status(ldx=15) == _lib.SEMX_ERR_SHAPE
    assert status(act=2) == _lib.SEMX_ERR_UNSUPPORTED
    assert status(w=None) == _lib.SEMX_ERR_NULL
    assert status(h=None) == _lib.SEMX_ERR_NULL
    assert status(x=4097, bf16=1) == _lib.SEMX_ERR_ALIGN
    assert status("semx_gated_linear_bwd") == _lib.SEMX_ERR_NULL
    assert status(rows=0) == _lib.SEMX_OK
    a = _lib.new_args(_lib.SemxGatedLinearArgs)
    a.rows, a.D, a.H = 5, 1000, 9
    assert lib.semx_gated_linear_saved_bytes(ctypes.byref(a)) == 2 * 5 * 16 * 4
    a.D, a.bf16 = 16, 1  # narrow: made again
    assert lib.semx_gated_linear_saved_bytes(ctypes.byref(a)) == 0


def test_factory_and_module():
    from semambaxlinoss_b200.gated_lru import GatedLruMixer
    from semambaxlinoss_b200.gated_mlp import GatedMLP
    from semambaxlinoss_b200.mamba_block import MambaBlock, create_block

    cfg = {"ssm": "gated_lru", "d_state": 4, "d_conv": 3, "expand": 2}
    block = create_block(16, dict(cfg, ssm_params={"rate_scale": 4.0}, mlp={"hidden_features": 24}))
    assert isinstance(block.mixer, GatedLruMixer) and block.mixer.rate_scale == 4.0 and block.mixer.d_conv == 3
    assert isinstance(block.mlp, GatedMLP) and block.mlp.fc1.weight.shape == (48, 16)
    assert create_block(16, cfg).mlp is None
    with pytest.raises(ValueError, match="causal"):
        create_block(16, dict(cfg, causal_conv=False))
    with pytest.raises(ValueError, match="feed-forward"):
        create_block(16, {"ssm": "hybrid", "mlp": {}, "backbone_1": cfg, "backbone_2": cfg})
    with pytest.raises(ValueError, match="activation"):
        GatedMLP(8, activation="relu")
    with pytest.raises(ValueError, match="decays"):
        GatedLruMixer(8, decay_min=0.0)
    torch.manual_seed(0)
    rate = GatedLruMixer(64).rate.detach().double()
    decay = torch.exp(-8 * torch.nn.functional.softplus(rate))
    assert bool(((decay > 0.8999) & (decay < 0.9991)).all())
    # Two residual branches per layer halve the variance of what each starts with.
    torch.manual_seed(1)
    both = MambaBlock(16, dict(cfg, mlp={"hidden_features": 400}, bidirectional=False)).forward_blocks[0]
    bound = (3 / 400) ** 0.5 * (2 / (1 + 5)) ** 0.5 / 2 ** 0.5
    assert 0.9 * bound < both.mlp.fc2.weight.abs().max() <= bound * 1.0001


def test_mixer_refuses_pool_arguments_without_a_cache():
    from semambaxlinoss_b200.gated_lru import GatedLruMixer

    with pytest.raises(ValueError, match="without a cache"):
        GatedLruMixer(8)(torch.zeros(1, 2, 8), slots=torch.zeros(1, dtype=torch.int32))


def test_recurrence_oracle_against_autograd():
    g = gen(0)
    rows, C, cu = 30, 5, [1, 10, 10, 28]
    x, r, i, z, dy = (randn((rows, C), g) for _ in range(5))
    rate, rb, ib = randn((C,), g) - 3, randn((C,), g), randn((C,), g)
    ins = [t.requires_grad_() for t in (x, r, i, z, rate, rb, ib)]
    rho, iota, _, a, _, gain = ogl.parts(r, i, rate, rb, ib)
    ys = [torch.zeros(C, dtype=torch.float64)] * rows
    for s in range(3):
        h = torch.zeros(C, dtype=torch.float64)
        for t in range(cu[s], cu[s + 1]):
            h = a[t] * h + gain[t] * iota[t] * x[t]
            ys[t] = h * torch.nn.functional.silu(z[t])
    grads = torch.autograd.grad(torch.stack(ys), ins, dy)
    out = ogl.scan(*(t.detach() for t in (x, r, i, rate)), cu, z.detach(), rb.detach(), ib.detach(), dy=dy)
    for name, q in zip(("dx", "dr", "di", "dz", "drate", "dr_bias", "di_bias"), grads):
        assert (out[name] - q).abs().max() < 1e-12, name


@pytest.mark.parametrize("kind", ["silu", "gelu"])
def test_projection_oracle_against_autograd(kind):
    g = gen(1)
    x, w, b, dh = randn((7, 6), g), randn((10, 6), g), randn((10,), g), randn((7, 5), g)
    ins = [t.requires_grad_() for t in (x, w, b)]
    u, v = torch.nn.functional.linear(x, w, b).chunk(2, -1)
    h = u * (torch.nn.functional.silu(v) if kind == "silu" else torch.nn.functional.gelu(v))
    grads = torch.autograd.grad(h, ins, dh)
    out = ogm.gated(x.detach(), w.detach(), b.detach(), kind, dh)
    assert (out["h"][0] - h).abs().max() < 1e-12
    for name, q in zip(("dx", "dw", "db"), grads):
        assert (out[name][0] - q).abs().max() < 1e-12, name
