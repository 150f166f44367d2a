"""Gated projection of a feed-forward block (``semx_gated_linear_fwd/bwd``) and the block's module.

    [u | g] = x W^T + b        h = u act(g)

* :func:`gated_linear` — the operator: both projections, the activation and the product in one
  kernel on the tensor cores, with gradients for every input. fp32 arithmetic on bf16 or fp32 operands.
* :class:`GatedMLP` — the module, ``fc2(gated_linear(x, fc1))``; ``create_block`` builds it where the
  configuration has ``mlp``.

CUDA tensors only, like the other operators of this package (RuntimeError otherwise).
"""
from __future__ import annotations

import torch
from torch import nn

from . import _lib
from .selective_state._batch import TYPES, check_same, rows_of

_ACTIVATIONS = {"silu": 0, "gelu": 1}


def _args(x, weight, bias, act):
    """The argument struct of x (rows, D) at any row stride."""
    a = _lib.new_args(_lib.SemxGatedLinearArgs)
    a.bf16, a.act = x.dtype == torch.bfloat16, act
    a.rows, a.D, a.H = x.shape[0], x.shape[1], weight.shape[0] // 2
    a.ldx = x.stride(0) if x.shape[0] > 1 else x.shape[1]
    a.x, a.w = x.data_ptr(), weight.data_ptr()
    if bias is not None:
        a.bias, a.bias_bf16 = bias.data_ptr(), bias.dtype == torch.bfloat16
    return a


def _workspace(a, backward, like):
    nbytes = _lib.load().semx_gated_linear_workspace_bytes(a, backward)
    ws = _lib.scratch(nbytes, like) if nbytes else None
    a.workspace = _lib.ptr(ws)
    return ws


def _forward(x, weight, bias, act, keep):
    """(h, u and g in front of the activation where ``keep``)."""
    a = _args(x, weight, bias, act)
    h = x.new_empty((a.rows, a.H))
    nbytes = _lib.load().semx_gated_linear_saved_bytes(a) if keep else 0
    saved = _lib.scratch(nbytes, x) if nbytes else None
    a.h, a.saved = h.data_ptr(), _lib.ptr(saved)
    ws = _workspace(a, 0, x)
    _lib.call("semx_gated_linear_fwd", a, x.device)
    return h, saved


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, act):
        w = weight.contiguous()
        b = None if bias is None else bias.contiguous()
        h, saved = _forward(x, w, b, act, True)
        ctx.save_for_backward(x, w, b, saved)
        ctx.cfg = (act, None if bias is None else bias.dtype)
        return h

    @staticmethod
    @_lib.once_differentiable
    def backward(ctx, dh):
        x, weight, bias, saved = ctx.saved_tensors
        act, bias_t = ctx.cfg
        need = ctx.needs_input_grad
        a = _args(x, weight, bias, act)
        dh = _lib.as_rows(dh, x.dtype)
        dx = x.new_empty(x.shape) if need[0] else None
        dw = torch.empty_like(weight) if need[1] else None
        db = weight.new_empty(weight.shape[0], dtype=torch.float32) if bias_t is not None and need[2] else None
        a.saved, a.dh, a.dx, a.dw, a.db = _lib.ptr(saved), dh.data_ptr(), _lib.ptr(dx), _lib.ptr(dw), _lib.ptr(db)
        ws = _workspace(a, 1, x)
        _lib.call("semx_gated_linear_bwd", a, x.device)
        return dx, dw, _lib.cast(db, bias_t), None


def gated_linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
                 activation: str = "silu") -> torch.Tensor:
    """``h = u act(g)`` with ``[u | g] = x weight^T + bias``: x (..., D), weight (2 H, D) (the value's
    rows, then the gate's, as one ``nn.Linear``), bias (2 H,) -> h (..., H) of x's type.

    x and weight are of one type, bf16 or fp32; bf16 autocast casts both. activation: "silu" or "gelu"
    (with the normal distribution). Sums are fp32; fp32 operands keep fp32's precision (an infinity
    among them gives NaN). With gradients wanted the forward keeps u and g in fp32 (8 bytes per element
    of h); in bf16 with x of up to 512 features the backward makes them again instead."""
    op = "gated_linear"
    if not x.is_cuda:
        raise RuntimeError(f"{op} requires CUDA tensors.")
    if activation not in _ACTIVATIONS:
        raise ValueError(f"{op}: activation must be 'silu' or 'gelu', got {activation!r}")
    if torch.is_autocast_enabled("cuda"):
        t = torch.get_autocast_dtype("cuda")
        if x.dtype in TYPES and weight.dtype in TYPES:
            x, weight = x.to(t), weight.to(t)
    if x.dtype not in TYPES:
        raise ValueError(f"{op}: unsupported dtype {x.dtype}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{op}: x must be (..., features), got {tuple(x.shape)}")
    D, dev = x.shape[-1], x.get_device()
    if weight.dim() != 2 or weight.shape[0] < 2 or weight.shape[0] % 2:
        raise ValueError(f"{op}: weight must be (2 hidden, {D}), got {tuple(weight.shape)}")
    check_same(op, "weight", weight, (weight.shape[0], D), (x.dtype,), dev)
    if bias is not None:
        check_same(op, "bias", bias, (weight.shape[0],), TYPES, dev)
    if _lib.in_dual_level():
        _lib.refuse_tangents(op, x, weight, bias)
    act = _ACTIVATIONS[activation]
    lead = x.shape[:-1]
    rows = x.reshape(-1, D) if x.dim() != 2 else x
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad
                                    or (bias is not None and bias.requires_grad)):
        rows = rows if rows_of(rows, D)[0] is rows else rows.contiguous()
        h = _GatedLinear.apply(rows, weight, bias, act)
    else:
        h, _ = _forward(rows_of(rows, D)[0], weight.contiguous(), None if bias is None else bias.contiguous(), act, False)
    return h if x.dim() == 2 else h.view(lead + (h.shape[-1],))


class GatedMLP(nn.Module):
    """Feed-forward half of a block: ``fc2(u act(g))`` with ``[u | g] = fc1(x)``, of (..., in_features).

    Args:
        in_features: input and output width.
        hidden_features: width of u and g. Default 8/3 of in_features, up to a multiple of 128.
        activation: "silu" (default) or "gelu".
        bias: biases of both projections. Default False.
    """

    def __init__(self, in_features: int, hidden_features: int | None = None, activation: str = "silu",
                 bias: bool = False):
        super().__init__()
        if activation not in _ACTIVATIONS:
            raise ValueError(f"GatedMLP: activation must be 'silu' or 'gelu', got {activation!r}")
        if hidden_features is None:
            hidden_features = -(-(8 * in_features // 3) // 128) * 128
        self.in_features, self.hidden_features, self.activation = in_features, hidden_features, activation
        self.fc1 = nn.Linear(in_features, 2 * hidden_features, bias=bias)
        self.fc2 = nn.Linear(hidden_features, in_features, bias=bias)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return self.fc2(gated_linear(x, self.fc1.weight, self.fc1.bias, activation=self.activation))
