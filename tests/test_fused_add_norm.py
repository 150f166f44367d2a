"""Blocks of ``create_block(rms_norm=False, fused_add_norm=True)`` take every tensor that the same
blocks with ``nn.LayerNorm`` take: what the layer norm kernel does not (CPU, fp16, fp64, rows of
more than 8192 elements, a residual that is broadcast, forward-mode tangents) gives the
same bits as theirs; what it does is within fp32 rounding of them."""
from __future__ import annotations

import pytest
import torch
from torch import nn

from semambaxlinoss_b200.layer_norm import LayerNorm
from semambaxlinoss_b200.mamba_block import Block, HybridBlock, create_block

CFG = {"ssm": "selective_lru", "d_state": 4, "d_conv": 4, "expand": 2}


class Pass(nn.Module):
    """In the mixer's place: the norm's output as it is."""

    def forward(self, x, inference_params=None):
        return x


def _pair(d, dtype=torch.float32, device="cpu", mlp=False):
    """The fused block and the one it stands for, with the same parameters."""
    def make(norm, fused):
        return Block(d, lambda _: Pass(), (lambda _: Pass()) if mlp else nn.Identity, norm_cls=norm, fused_add_norm=fused)

    fused, plain = make(LayerNorm, True), make(nn.LayerNorm, False)
    with torch.no_grad():
        for p in fused.parameters():
            p.add_(torch.randn(p.shape) * 0.1)
    plain.load_state_dict(fused.state_dict())
    return fused.to(device, dtype), plain.to(device, dtype)


def _same(d, dtypes, device="cpu", param=torch.float32, residual_shape=None, mlp=False):
    fused, plain = _pair(d, param, device, mlp)
    fired = []
    fused.norm.register_forward_hook(lambda *a: fired.append(1))
    x = torch.randn(3, 5, d).to(device, dtypes[0])
    r = None if dtypes[1] is None else torch.randn(residual_shape or x.shape).to(device, dtypes[1])
    results = []
    for block in (fused, plain):
        leaves = [t.clone().requires_grad_() for t in (x, r) if t is not None]
        y, s = block(*leaves)
        grads = torch.autograd.grad((y.float().square().sum() + s.float().sum()), leaves + list(block.parameters()))
        results.append((y, s) + grads)
    assert fired == [1]
    for p, q in zip(*results):
        assert p.dtype == q.dtype and torch.equal(p, q)


def test_is_an_nn_layer_norm():
    block = create_block(8, CFG, rms_norm=False, fused_add_norm=True)
    plain = create_block(8, CFG, rms_norm=False)
    assert isinstance(block.norm, nn.LayerNorm) and type(plain.norm) is nn.LayerNorm
    assert block.norm.normalized_shape == plain.norm.normalized_shape and block.norm.eps == plain.norm.eps
    assert list(block.state_dict()) == list(plain.state_dict())


@pytest.mark.parametrize("dtypes,param", [((torch.float32, None), torch.float32), ((torch.float32,) * 2, torch.float32),
                                          ((torch.float64,) * 2, torch.float64), ((torch.float16, torch.float32), torch.float32),
                                          ((torch.bfloat16, None), torch.bfloat16)])
@pytest.mark.parametrize("mlp", [False, True])
def test_cpu_tensors(dtypes, param, mlp):
    _same(12, dtypes, param=param, mlp=mlp)


def test_hybrid_block_on_the_cpu():
    torch.manual_seed(0)
    blocks = [HybridBlock(8, Pass(), Pass(), "sequential", norm_cls=n) for n in (LayerNorm, nn.LayerNorm)]
    blocks[1].load_state_dict(blocks[0].state_dict())
    x = torch.randn(2, 3, 8)
    for p, q in zip(blocks[0](x, x + 1), blocks[1](x, x + 1)):
        assert torch.equal(p, q)


def test_tangents_on_the_cpu():
    from torch.autograd import forward_ad

    fused, plain = _pair(8)
    x, r, t = torch.randn(3, 8), torch.randn(3, 8), torch.randn(3, 8)
    with forward_ad.dual_level(), torch.no_grad():
        d = forward_ad.make_dual(x, t)
        for p, q in zip(fused(d, r), plain(d, r)):
            assert torch.equal(forward_ad.unpack_dual(p).tangent, forward_ad.unpack_dual(q).tangent)


@pytest.mark.gpu
@pytest.mark.parametrize("d,dtypes,param,shape", [
    (12, (torch.float16, None), torch.float16, None), (12, (torch.float16, torch.float32), torch.float32, None),
    (12, (torch.float64,) * 2, torch.float64, None), (12, (torch.float32, torch.float64), torch.float32, None),
    (32776, (torch.float32,) * 2, torch.float32, None), (8200, (torch.float32,) * 2, torch.float32, None), (12, (torch.float32,) * 2, torch.float32, (5, 12)),
    (12, (torch.bfloat16, torch.float16), torch.bfloat16, None)])
def test_what_the_kernel_does_not_take(d, dtypes, param, shape):
    _same(d, dtypes, "cuda", param, shape)


@pytest.mark.gpu
def test_tangents():
    from torch.autograd import forward_ad

    fused, plain = _pair(16, device="cuda")
    x, r, t = (torch.randn(3, 16, device="cuda") for _ in range(3))
    with forward_ad.dual_level(), torch.no_grad():
        d = forward_ad.make_dual(r, t)
        for p, q in zip(fused(x, d), plain(x, d)):
            assert torch.equal(forward_ad.unpack_dual(p).tangent, forward_ad.unpack_dual(q).tangent)


@pytest.mark.gpu
@pytest.mark.parametrize("xt,rt,param", [(torch.float32, torch.float32, torch.float32), (torch.bfloat16, torch.float32, torch.float32),
                                         (torch.bfloat16, None, torch.float32), (torch.float32, torch.bfloat16, torch.float32)])
def test_what_the_kernel_takes(xt, rt, param):
    """The norm of the same sum in fp32 by two ways: each value is a sum of a few terms of the size of
    the largest, 64 steps of 2^-24 of it cover both."""
    fused, plain = _pair(200, param, "cuda", mlp=True)
    x = torch.randn(7, 200, device="cuda").to(xt)
    r = None if rt is None else torch.randn(7, 200, device="cuda").to(rt)
    with torch.no_grad():
        for p, q in zip(fused(x, r), plain(x, r)):
            assert p.dtype == q.dtype
            assert (p - q).abs().max() <= 64 * 2.0 ** -24 * (1 + q.abs().max())
