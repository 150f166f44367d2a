"""Short causal depthwise convolution over sequences that can keep their last inputs
(``semx_short_conv_fwd/bwd``).

    y[t, c] = act(bias[c] + sum_k weight[c, k] x[t - (K - 1) + k, c])

Unlike the convolution inside ``MambaStyleMixer`` (:mod:`semambaxlinoss_b200.mixer`), x is
any tensor of rows (packed sequences of many lengths too), y has x's type, and a sequence
can start from the window that an earlier call left.
"""
from __future__ import annotations

import torch

from .. import _lib
from ._batch import TYPES, batch, check_same, rows_of, set_pool

_ACTIVATIONS = {"silu": 1, None: 0}


def _weight(op, weight, C):
    """(C, K) of a weight (C, K) or (C, 1, K) (``nn.Conv1d``'s, groups = channels)."""
    w = weight.squeeze(1) if weight.dim() == 3 and weight.shape[1] == 1 else weight
    shape = w.shape
    if len(shape) != 2 or shape[0] != C or not 1 <= shape[1] <= 8:
        raise ValueError(f"{op}: weight must be ({C}, taps) or ({C}, 1, taps) with 1 to 8 taps, got "
                         f"{tuple(weight.shape)}")
    return w


def _args(x, w, b, silu, S, rows, L, cu):
    C = x.shape[-1]
    xr, ld = rows_of(x, C)
    a = _lib.new_args(_lib.SemxShortConvArgs)
    a.K, a.silu, a.bf16 = w.shape[1], silu, x.dtype == torch.bfloat16
    a.S, a.rows, a.L, a.C, a.ldx = S, rows, L, C, ld
    a.x, a.w = xr.data_ptr(), w.data_ptr()
    if b is not None:
        a.b = b.data_ptr()
    if cu is not None:
        a.cu_seqlens = cu.data_ptr()
    return a, xr


class _ShortConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, silu, S, rows, L, cu):
        w, b = _lib.param32(weight), _lib.param32(bias)
        a, xr = _args(x, w, b, silu, S, rows, L, cu)
        y = x.new_empty(x.shape)
        a.y = y.data_ptr()
        _lib.call("semx_short_conv_fwd", a, x.device)
        ctx.save_for_backward(xr, w, b, cu)
        ctx.cfg = (silu, S, rows, L, weight.dtype, None if bias is None else bias.dtype)
        return y

    @staticmethod
    @_lib.once_differentiable
    def backward(ctx, dy):
        x, w, b, cu = ctx.saved_tensors
        silu, S, rows, L, wdt, bdt = ctx.cfg
        a, xr = _args(x, w, b, silu, S, rows, L, cu)
        dy = _lib.as_rows(dy, x.dtype)
        dx = x.new_empty(x.shape)
        dw = torch.empty_like(w) if ctx.needs_input_grad[1] else None
        db = torch.empty_like(b) if b is not None and ctx.needs_input_grad[2] else None
        a.dy, a.dx, a.dw, a.db = dy.data_ptr(), dx.data_ptr(), _lib.ptr(dw), _lib.ptr(db)
        ws = None
        if dw is not None or db is not None:
            ws = _lib.scratch(_lib.load().semx_short_conv_workspace_bytes(a), x)
            a.workspace = ws.data_ptr()
        _lib.call("semx_short_conv_bwd", a, x.device)
        return dx, _lib.cast(dw, wdt), _lib.cast(db, bdt), None, None, None, None, None


def _silu_flag(op, activation):
    if activation not in _ACTIVATIONS:
        raise ValueError(f"{op}: activation must be 'silu' or None, got {activation!r}")
    return _ACTIVATIONS[activation]


def short_conv(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, activation: str | None = "silu",
               cu_seqlens: torch.Tensor | None = None, state: torch.Tensor | None = None,
               slots: torch.Tensor | None = None, fresh: torch.Tensor | None = None) -> torch.Tensor:
    """Causal depthwise convolution of the sequences in ``x``; y has x's shape and type.

    x: (S, L, C), or packed (rows, C) with ``cu_seqlens`` (S + 1, int32): sequence s owns rows
    cu_seqlens[s] .. cu_seqlens[s+1] - 1 (none, if they are equal); rows in front of cu_seqlens[0]
    and from cu_seqlens[S] on belong to no sequence and come out as zeros. Rows may lie at any stride (a slice of
    the in_proj output is read in place). weight (C, K) or (C, 1, K), K from 1 to 8, bias (C,).

    Training: gradients flow to x, weight and bias, every sequence starts from zeros.
    Prompts: ``state`` (entries, K - 1, C) in x's type holds the last K - 1 inputs of running
    sequences and is updated in place; sequence s uses entry ``slots[s]`` (int32; entry s
    without slots), from zeros where ``fresh[s]``. A negative slot: no entry, from zeros. A
    slot behind the pool, or one an earlier sequence of the call has, gives NaN for that
    sequence and leaves the entry alone. Not differentiable: refused while a gradient is
    wanted (call it under ``torch.no_grad()``)."""
    op = "short_conv"
    S, rows, L = batch(op, x, cu_seqlens)
    return _run(op, x, weight, bias, activation, S, rows, L, cu_seqlens, state, slots, fresh)


def _run(op, x, weight, bias, activation, S, rows, L, cu_seqlens, state, slots, fresh):
    silu = _silu_flag(op, activation)
    if _lib.in_dual_level():
        _lib.refuse_tangents(op, x, weight, bias, state)
    C, dev = x.shape[-1], x.get_device()
    w = _weight(op, weight, C)
    if w.dtype not in TYPES or w.get_device() != dev:
        check_same(op, "weight", w, w.shape, TYPES, dev)
    if bias is not None:
        check_same(op, "bias", bias, (C,), TYPES, dev)
    if torch.is_grad_enabled() and (x.requires_grad or w.requires_grad or (bias is not None and bias.requires_grad)):
        if state is not None:
            raise ValueError(f"{op}: a state is for inference; the call wants gradients")
        if slots is not None or fresh is not None:
            raise ValueError(f"{op}: slots / fresh without a state")
        return _ShortConv.apply(x, w, bias, silu, S, rows, L, cu_seqlens)
    w, bias = _lib.param32(w), _lib.param32(bias)
    a, xr = _args(x, w, bias, silu, S, rows, L, cu_seqlens)
    K = w.shape[1]
    if K > 1 or state is None:  # one tap keeps nothing
        set_pool(op, a, S, dev, state, (K - 1, C), x.dtype, slots, fresh)
    y = x.new_empty(x.shape)
    a.y = y.data_ptr()
    _lib.call("semx_short_conv_fwd", a, x.device)
    return y


def short_conv_step(x: torch.Tensor, state: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
                    activation: str | None = "silu", slots: torch.Tensor | None = None) -> torch.Tensor:
    """One token of every sequence: x (S, C) -> y (S, C); the windows in ``state`` (entries,
    K - 1, C) move on by one in place. Slots as in :func:`short_conv`."""
    op = "short_conv_step"
    if not x.is_cuda:
        raise RuntimeError(f"{op} requires CUDA tensors.")
    if x.dim() != 2 or x.dtype not in TYPES:
        raise ValueError(f"{op}: x must be fp32 or bf16 (sequences, channels), got {x.dtype} {tuple(x.shape)}")
    if state is None:
        raise ValueError(f"{op}: a state is needed")
    S = x.shape[0]
    return _run(op, x, weight, bias, activation, S, S, 1, None, state, slots, None)
