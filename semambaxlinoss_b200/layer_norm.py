"""Layer normalisation with an optional residual added first (``semx_layer_norm_fwd/bwd``).

* :func:`layer_norm` — the operator: ``s = x + residual`` (``x`` when there is none),
  ``y = (s - mean(s)) / sqrt(var(s) + eps) * weight + bias`` over the last dimension, in
  fp32 arithmetic, with gradients for every input.
* :class:`LayerNorm` — the module: parameters, names and initial values of
  ``nn.LayerNorm(d, eps)``, which it is, forward through the operator. ``create_block`` builds it with
  ``rms_norm=False, fused_add_norm=True``, and the pre-norm ``Block`` then runs its
  residual add and its norm as one kernel.

CUDA tensors only, like the other operators of this package (RuntimeError otherwise);
fp32 and bf16; rows of up to 32768 elements.
"""
from __future__ import annotations

import torch
from torch import nn

from . import _lib

_TYPES = (torch.float32, torch.bfloat16)
# Widest rows that a block's fused add and norm takes. Wider ones spill (a row has 1024 threads at most): 4096
# rows of 16384, training pass of add and norm with an fp32 residual, 969 us, as nn.LayerNorm behind an
# addition 707; 8192 rows of 8192, 413 and 664.
BLOCK_WIDTH = 8192


def _forward(x, weight, bias, eps, residual, out_dtype, stats):
    """Runs the forward; returns (y, s, kept): kept (2 rows) holds mean and 1 / sqrt(var + eps)
    where ``stats``, else None."""
    d = x.shape[-1]
    x = x.contiguous()
    y = torch.empty_like(x, dtype=out_dtype)
    a = _lib.new_args(_lib.SemxLayerNormArgs)
    a.eps, a.n, a.d = eps, x.numel() // d, d
    a.x_bf16, a.y_bf16 = x.dtype == torch.bfloat16, out_dtype == torch.bfloat16
    a.x, a.y = x.data_ptr(), y.data_ptr()
    s = x
    if residual is not None:
        residual = residual.contiguous()
        s = torch.empty_like(residual if x.dtype == torch.bfloat16 else x)  # the wider type
        a.r_bf16, a.s_bf16 = residual.dtype == torch.bfloat16, s.dtype == torch.bfloat16
        a.residual, a.sum = residual.data_ptr(), s.data_ptr()
    if weight is not None:
        a.weight = weight.data_ptr()
    if bias is not None:
        a.bias = bias.data_ptr()
    kept = None
    if stats:
        kept = x.new_empty(2 * a.n, dtype=torch.float32)
        at = kept.data_ptr()
        a.mean, a.rstd = at, at + 4 * a.n
    _lib.call("semx_layer_norm_fwd", a, x.device)
    return y, s, kept


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, residual, out_dtype):
        ctx.set_materialize_grads(False)
        w = _lib.param32(weight)
        y, s, kept = _forward(x, w, _lib.param32(bias), eps, residual, out_dtype, True)
        ctx.save_for_backward(s, w, kept)
        ctx.cfg = (eps, out_dtype, x.dtype, None if residual is None else residual.dtype,
                   None if weight is None else weight.dtype, None if bias is None else bias.dtype)
        return y if residual is None else (y, s)

    @staticmethod
    @_lib.once_differentiable
    def backward(ctx, dy, dsum=None):
        s, w, kept = ctx.saved_tensors
        eps, ydt, xdt, rdt, wdt, bdt = ctx.cfg
        if dy is None and dsum is None:
            return None, None, None, None, None, None
        shape = s.shape
        d = shape[-1]
        dy = s.new_zeros(shape, dtype=ydt) if dy is None else _lib.as_rows(dy, ydt)
        dsum = None if dsum is None else _lib.as_rows(dsum, s.dtype)
        dx = torch.empty_like(s, dtype=xdt)
        a = _lib.new_args(_lib.SemxLayerNormArgs)
        a.eps, a.n, a.d = eps, kept.shape[0] // 2, d
        a.x_bf16, a.y_bf16, a.s_bf16 = xdt == torch.bfloat16, ydt == torch.bfloat16, s.dtype == torch.bfloat16
        at = kept.data_ptr()
        a.sum, a.mean, a.rstd, a.weight = s.data_ptr(), at, at + 4 * a.n, _lib.ptr(w)
        a.dy, a.dsum, a.dx = dy.data_ptr(), _lib.ptr(dsum), dx.data_ptr()
        need = ctx.needs_input_grad
        dr = dx if rdt == xdt else None
        if rdt is not None and need[4] and dr is None:
            dr = torch.empty_like(s, dtype=rdt)
            a.r_bf16, a.dresidual = rdt == torch.bfloat16, dr.data_ptr()
        dw = s.new_empty(d, dtype=torch.float32) if wdt is not None and need[1] else None
        db = s.new_empty(d, dtype=torch.float32) if bdt is not None and need[2] else None
        ws = None
        if dw is not None or db is not None:
            a.dweight, a.dbias = _lib.ptr(dw), _lib.ptr(db)
            ws = _lib.scratch(_lib.load().semx_layer_norm_workspace_bytes(a), s)
            a.workspace = ws.data_ptr()
        _lib.call("semx_layer_norm_bwd", a, s.device)
        return (dx, _lib.cast(dw, wdt), _lib.cast(db, bdt), None, dr if rdt is not None else None, None)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None, bias: torch.Tensor | None = None, eps: float = 1e-5,
               residual: torch.Tensor | None = None, out_dtype: torch.dtype | None = None):
    """Layer norm of the last dimension of ``x`` (..., d); with ``residual`` (x's shape) of
    their sum, which is returned too, in the wider of the two types.

    ``weight`` and ``bias`` (d,) may be None. ``out_dtype``: the type of y (x's by default).
    Returns ``y``, or ``(y, s)`` with a residual. Gradients flow to x, residual, weight and
    bias, from y and from s; the gradients of weight and bias are reduced over rows in a
    fixed order. A row of the backward costs no recomputation: mean and 1 / sqrt(var + eps)
    are kept in fp32."""
    if not x.is_cuda:
        raise RuntimeError("layer_norm requires CUDA tensors.")
    out_dtype = x.dtype if out_dtype is None else out_dtype
    if x.dtype not in _TYPES or out_dtype not in _TYPES:
        raise ValueError(f"layer_norm: unsupported dtype {x.dtype if x.dtype not in _TYPES else out_dtype}")
    d = x.shape[-1] if x.dim() else 0
    if d < 1:
        raise ValueError(f"layer_norm: nothing to normalise in shape {tuple(x.shape)}")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is not None and (p.shape != (d,) or p.get_device() != x.get_device()):
            raise ValueError(f"layer_norm: {name} must be ({d},) on {x.device}, got {tuple(p.shape)} on {p.device}")
    if residual is not None and (residual.shape != x.shape or residual.get_device() != x.get_device()
                                 or residual.dtype not in _TYPES):
        raise ValueError(f"layer_norm: residual must be fp32 or bf16 {tuple(x.shape)} on {x.device}, got "
                         f"{residual.dtype} {tuple(residual.shape)} on {residual.device}")
    if _lib.in_dual_level():
        _lib.refuse_tangents("layer_norm", x, weight, bias, residual)
    eps = float(eps)
    if torch.is_grad_enabled() and (
            x.requires_grad or (weight is not None and weight.requires_grad) or (bias is not None and bias.requires_grad)
            or (residual is not None and residual.requires_grad)):
        return _LayerNorm.apply(x, weight, bias, eps, residual, out_dtype)
    y, s, _ = _forward(x, _lib.param32(weight), _lib.param32(bias), eps, residual, out_dtype, False)
    return y if residual is None else (y, s)


class LayerNorm(nn.LayerNorm):
    """``nn.LayerNorm`` over the last dimension, with its parameters and state dict, through
    :func:`layer_norm`. ``forward(x, residual)`` adds the residual first and returns
    (y, x + residual)."""

    def __init__(self, hidden_size: int, eps: float = 1e-5, device=None, dtype=None):
        super().__init__(hidden_size, eps, device=device, dtype=dtype)

    def takes(self, x: torch.Tensor, residual: torch.Tensor | None = None) -> bool:
        """Whether ``self(x, residual, out_dtype=weight.dtype)`` is a call of the operator's."""
        w = self.weight
        return (x.is_cuda and x.dtype in _TYPES and w.dtype in _TYPES and w.get_device() == x.get_device()
                and w.shape[0] <= BLOCK_WIDTH and not _lib.has_tangents(x, residual, w, self.bias)
                and (residual is None or (residual.dtype in _TYPES and residual.shape == x.shape
                                          and residual.get_device() == x.get_device())))

    def add(self, x: torch.Tensor, residual: torch.Tensor | None = None):
        """(the norm of x + residual in the weight's type, x + residual), in one kernel where the
        operator takes the tensors, else as ``nn.LayerNorm`` behind an addition."""
        dtype = self.weight.dtype
        if residual is None:
            rows = x.to(dtype=dtype)
            return self(rows, plain=not self.takes(rows)), x
        if self.takes(x, residual):
            return self(x, residual, out_dtype=dtype)
        residual = x + residual
        return self(residual.to(dtype=dtype), plain=True), residual

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None, out_dtype: torch.dtype | None = None,
                plain: bool = False):
        if plain:  # as nn.LayerNorm, for what the operator does not take (see add)
            return super().forward(x)
        return layer_norm(x, self.weight, self.bias, self.eps, residual, out_dtype)
