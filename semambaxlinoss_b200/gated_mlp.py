"""Gated projection of a feed-forward block (``semx_gated_linear_fwd/bwd``) and the block's module.

    [u | g] = x W^T + b        h = u act(g)

* :func:`gated_linear` — the operator: both projections, the activation and the product in one
  kernel on the tensor cores, with gradients for every input. fp32 arithmetic on bf16 or fp32 operands.
* :class:`GatedMLP` — the module, ``fc2(gated_linear(x, fc1))``; ``create_block`` builds it where the
  configuration has ``mlp``.

CUDA tensors only, like the other operators of this package (RuntimeError otherwise).
"""
from __future__ import annotations

import functools

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


@functools.lru_cache(maxsize=256)
def _sizes(rows, D, H, ldx, bf16, x_odd, w_odd, backward, dx, dw, db):
    """Bytes of what the forward keeps, and of a call's workspace: the library's, by its sizes, whether x
    and w lie on 16 bytes, and the gradients that are wanted."""
    a = _lib.new_args(_lib.SemxGatedLinearArgs)
    a.bf16, a.rows, a.D, a.H, a.ldx = bf16, rows, D, H, ldx
    a.x, a.w, a.h, a.dh, a.saved = 256 + x_odd, 256 + w_odd, 256, 256, 256
    a.dx, a.dw, a.db = 256 * dx or None, 256 * dw or None, 256 * db or None
    lib = _lib.load()
    return lib.semx_gated_linear_saved_bytes(a), lib.semx_gated_linear_workspace_bytes(a, backward)


def _sizes_of(a, backward):
    return _sizes(a.rows, a.D, a.H, a.ldx, a.bf16, a.x % 16, a.w % 16, backward, bool(a.dx), bool(a.dw), bool(a.db))


def _workspace(a, nbytes, like):
    if not nbytes:
        return None
    ws = _lib.scratch(nbytes, like)
    a.workspace, a.workspace_bytes = ws.data_ptr(), nbytes
    return ws


def _forward(x, weight, bias, act, keep):
    """(h, u and g in front of the activation where ``keep``)."""
    a = _args(x, weight, bias, act)
    h = x.new_empty((a.rows, a.H))
    if a.rows == 0:
        return h, None
    kept, nbytes = _sizes_of(a, 0)
    saved = _lib.scratch(kept, x) if keep and kept else None
    a.h, a.saved = h.data_ptr(), _lib.ptr(saved)
    ws = _workspace(a, nbytes, x)
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
        # Hooks on saved tensors may have brought them back laid out otherwise.
        x, weight = rows_of(x, x.shape[1])[0], weight.contiguous()
        a = _args(x, weight, bias, act)
        dh = _lib.as_rows(dh, x.dtype)
        dx = x.new_empty(x.shape) if need[0] else None
        dw = torch.empty_like(weight) if need[1] else None
        db = weight.new_empty(weight.shape[0], dtype=torch.float32) if bias_t is not None and need[2] else None
        a.saved, a.dh, a.dx, a.dw, a.db = _lib.ptr(saved), dh.data_ptr(), _lib.ptr(dx), _lib.ptr(dw), _lib.ptr(db)
        ws = _workspace(a, _sizes_of(a, 1)[1], x) if a.rows else None
        _lib.call("semx_gated_linear_bwd", a, x.device)
        return dx, dw, _lib.cast(db, bias_t), None


def gated_linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
                 activation: str = "silu") -> torch.Tensor:
    """``h = u act(g)`` with ``[u | g] = x weight^T + bias``: x (..., D), weight (2 H, D) (the value's
    rows, then the gate's, as one ``nn.Linear``), bias (2 H,) -> h (..., H) of x's type.

    x and weight are of one type, bf16 or fp32; bf16 autocast casts both. activation: "silu" or "gelu"
    (with the normal distribution). Sums are fp32, and fp32 operands keep fp32's precision; an infinity
    among fp32 operands makes what depends on it infinite or NaN, from 17 rows on always NaN. With bf16
    operands the backward rounds the gradients of u and g to bf16 before it multiplies them with the
    weights and x, as layers in bf16 do (dx and dW are 0.0023 off instead of the 0.0017 of their own
    rounding); u, g and the activation are not rounded. With gradients wanted the forward keeps u and g in
    fp32 (8 bytes per element of h); in bf16 with x of up to 512 features the backward makes them again
    instead."""
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
        h = _forward(rows_of(rows, D)[0], weight.contiguous(), None if bias is None else bias.contiguous(), act, False)[0]
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
