"""Blocks with the gated recurrence or a feed-forward half inside MambaBlock and TFMambaBlock: behind mixers that
read token layouts in place, and behind those that do not, both directions, against the same modules called on
plain copies. Tolerances: fp32 operators that differ in the order of their sums only, 1e-4 of the largest value
(tests/parity.py)."""
from __future__ import annotations

import pytest
import torch

from tests.parity import assert_close, cuda, gen, randn

pytestmark = pytest.mark.gpu
B, T, F, C = 2, 37, 21, 32
BASE = {"d_state": 4, "d_conv": 4, "expand": 2}
MIXERS = {"gated_lru": {"ssm": "gated_lru"}, "selective_lru": {"ssm": "selective_lru", "ssm_params": {"dt_rank": 4}},
          "linoss": {"ssm": "linoss"}, "selective_state": {"ssm": "selective_state"}}


def _cfg(mixer, mlp, **kw):
    return dict(BASE, **MIXERS[mixer], **({} if mlp is None else {"mlp": mlp}), **kw)


def _one_direction(blocks, x):
    """Pre-norm blocks on plain (batch, length, channels) copies, spelled out."""
    h, res = x, None
    for b in blocks:
        res = h if res is None else h + res
        h = b.mixer(b.norm(res))
        if b.mlp is not None:
            res = h + res
            h = b.mlp.fc2(_gated(b.mlp, b.norm2(res)))
    return h + res


def _gated(mlp, x):
    u, g = mlp.fc1(x).chunk(2, -1)
    return u * (torch.nn.functional.silu(g) if mlp.activation == "silu" else torch.nn.functional.gelu(g))


def _mamba(m, x):
    y = _one_direction(m.forward_blocks, x)
    if not m.bidirectional:
        return y
    return torch.cat([y, torch.flip(_one_direction(m.backward_blocks, torch.flip(x, [1]).contiguous()), [1])], -1)


def _time_frequency(m, x):
    b, c, t, f = x.shape
    x = x.permute(0, 3, 2, 1).reshape(b * f, t, c)
    x = m._project(m.tlinear, _mamba(m.time_mamba, x)) + x
    x = x.view(b, f, t, c).permute(0, 2, 1, 3).reshape(b * t, f, c)
    x = m._project(m.flinear, _mamba(m.freq_mamba, x)) + x
    return x.view(b, t, f, c).permute(0, 3, 1, 2)


def _compare(m, run, plain, x, dy):
    params = list(m.parameters())
    out = []
    for f in (run, plain):
        v = x.clone().requires_grad_()
        y = f(v)
        out.append([y] + list(torch.autograd.grad(y, [v] + params, dy)))
    assert out[0][0].shape == out[1][0].shape
    for name, a, b in zip(["y", "dx"] + [n for n, _ in m.named_parameters()], *out):
        assert_close(a, b, 1e-4, name)


@pytest.mark.parametrize("time_mixer,freq_mixer", [("gated_lru", "gated_lru"), ("selective_lru", "gated_lru"),
                                                   ("gated_lru", "linoss"), ("selective_state", "selective_lru")])
@pytest.mark.parametrize("mlp", [None, {}, {"hidden_features": 50, "activation": "gelu", "bias": True}])
@pytest.mark.parametrize("bidirectional", [True, False])
def test_time_frequency_block(time_mixer, freq_mixer, mlp, bidirectional):
    from semambaxlinoss_b200.mamba_block import TFMambaBlock

    torch.manual_seed(3)
    cfg = {"model_cfg": dict(hid_feature=C, use_transpose=bidirectional,
                             time_mixer=_cfg(time_mixer, mlp, bidirectional=bidirectional),
                             freq_mixer=_cfg(freq_mixer, mlp, bidirectional=bidirectional))}
    m = TFMambaBlock(cfg).to(cuda())
    g = gen(4)
    x, dy = (randn((B, C, T, F), g).float().to(cuda()) for _ in range(2))
    _compare(m, m, lambda v: _time_frequency(m, v), x, dy)


@pytest.mark.parametrize("mixer", list(MIXERS))
@pytest.mark.parametrize("mlp", [None, {}, {"hidden_features": 50, "activation": "gelu", "bias": True}])
def test_mamba_block(mixer, mlp):
    from semambaxlinoss_b200.mamba_block import MambaBlock

    torch.manual_seed(5)
    m = MambaBlock(C, _cfg(mixer, mlp)).to(cuda())
    g = gen(6)
    x, dy = randn((B, T, C), g).float().to(cuda()), randn((B, T, 2 * C), g).float().to(cuda())
    _compare(m, m, lambda v: _mamba(m, v), x, dy)


@pytest.mark.parametrize("rms_norm,fused", [(True, False), (False, True), (False, False)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_block_norms_and_residual_types(rms_norm, fused, dtype):
    """Both norms, the fused addition, and a residual kept in fp32, with a feed-forward half."""
    from semambaxlinoss_b200.mamba_block import create_block

    for fp32 in (False, True):
        torch.manual_seed(7)
        block = create_block(C, _cfg("gated_lru", {}), rms_norm=rms_norm, fused_add_norm=fused, residual_in_fp32=fp32)
        block = block.to(cuda(), dtype)
        block.mixer.rate.data = block.mixer.rate.data.float()
        x = randn((B, T, C), gen(8)).to(dtype).to(cuda()).requires_grad_()
        h, res = block(x)
        assert h.dtype == dtype and res.dtype == (torch.float32 if fp32 else dtype)
        want = _one_direction([block], x)
        # bf16: each of some ten results on the way is rounded by 2^-8.
        assert_close((h + res).float(), want.float(), 1e-4 if dtype == torch.float32 else 4e-2)
        (h + res).float().sum().backward()
        assert torch.isfinite(x.grad).all() and x.grad.any()
