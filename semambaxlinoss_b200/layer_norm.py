"""Layer normalisation with an optional residual added first (``semx_layer_norm_fwd/bwd``).

* :func:`layer_norm` — the operator: ``s = x + residual`` (``x`` when there is none),
  ``y = (s - mean(s)) / sqrt(var(s) + eps) * weight + bias`` over the last dimension, in
  fp32 arithmetic, with gradients for every input.
* :class:`LayerNorm` — the module: parameters, names and initial values of
  ``nn.LayerNorm(d, eps)``, forward through the operator. ``create_block`` builds it with
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
MAX_WIDTH = 32768


def _param(p):
    if p is None or (p.dtype == torch.float32 and p.is_contiguous()):
        return p
    return p.detach().to(torch.float32).contiguous()


def _forward(x, weight, bias, eps, residual, out_dtype, stats):
    """Runs the forward on detached tensors; returns (y, s, mean, rstd), mean and rstd None
    unless ``stats``."""
    d = x.shape[-1]
    x = x.contiguous()
    y = x.new_empty(x.shape, dtype=out_dtype)
    a = _lib.new_args(_lib.SemxLayerNormArgs)
    a.eps, a.n, a.d = eps, x.numel() // d, d
    a.x_bf16, a.y_bf16 = x.dtype == torch.bfloat16, out_dtype == torch.bfloat16
    a.x, a.y = x.data_ptr(), y.data_ptr()
    s = x
    if residual is not None:
        residual = residual.contiguous()
        s = x.new_empty(x.shape, dtype=residual.dtype if x.dtype == torch.bfloat16 else x.dtype)
        a.r_bf16, a.s_bf16 = residual.dtype == torch.bfloat16, s.dtype == torch.bfloat16
        a.residual, a.sum = residual.data_ptr(), s.data_ptr()
    if weight is not None:
        a.weight = weight.data_ptr()
    if bias is not None:
        a.bias = bias.data_ptr()
    mean = rstd = None
    if stats:
        mean, rstd = torch.empty((2, a.n), dtype=torch.float32, device=x.device).unbind(0)
        a.mean, a.rstd = mean.data_ptr(), rstd.data_ptr()
    _lib.call("semx_layer_norm_fwd", a, x.device)
    return y, s, mean, rstd


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, residual, out_dtype):
        ctx.set_materialize_grads(False)
        w, b = _param(weight), _param(bias)
        r = residual
        y, s, mean, rstd = _forward(x, w, b, eps, r, out_dtype, True)
        ctx.save_for_backward(s, w, mean, rstd)
        ctx.cfg = (eps, out_dtype, x.dtype, None if r is None else r.dtype,
                   None if weight is None else weight.dtype, None if bias is None else bias.dtype)
        return y if r is None else (y, s)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dsum=None):
        s, w, mean, rstd = ctx.saved_tensors
        eps, ydt, xdt, rdt, wdt, bdt = ctx.cfg
        if dy is None and dsum is None:
            return None, None, None, None, None, None
        dev, d = s.device, s.shape[-1]
        dy = torch.zeros(s.shape, dtype=ydt, device=dev) if dy is None else dy.to(ydt).contiguous()
        dsum = None if dsum is None else dsum.to(s.dtype).contiguous()
        dx = torch.empty(s.shape, dtype=xdt, device=dev)
        a = _lib.new_args(_lib.SemxLayerNormArgs)
        a.eps, a.n, a.d = eps, s.numel() // d, d
        a.x_bf16, a.y_bf16, a.s_bf16 = xdt == torch.bfloat16, ydt == torch.bfloat16, s.dtype == torch.bfloat16
        a.sum, a.mean, a.rstd, a.weight = s.data_ptr(), mean.data_ptr(), rstd.data_ptr(), _lib.ptr(w)
        a.dy, a.dsum, a.dx = dy.data_ptr(), _lib.ptr(dsum), dx.data_ptr()
        dr = dx if rdt == xdt else None
        if rdt is not None and ctx.needs_input_grad[4] and dr is None:
            dr = torch.empty(s.shape, dtype=rdt, device=dev)
            a.r_bf16, a.dresidual = rdt == torch.bfloat16, dr.data_ptr()
        dw = torch.empty(d, dtype=torch.float32, device=dev) if wdt is not None and ctx.needs_input_grad[1] else None
        db = torch.empty(d, dtype=torch.float32, device=dev) if bdt is not None and ctx.needs_input_grad[2] else None
        ws = None
        if dw is not None or db is not None:
            a.dweight, a.dbias = _lib.ptr(dw), _lib.ptr(db)
            ws = _lib.empty_f32(_lib.load().semx_layer_norm_workspace_bytes(a), dev)
            a.workspace = ws.data_ptr()
        _lib.call("semx_layer_norm_bwd", a, dev)
        return (dx, None if dw is None else dw.to(wdt), None if db is None else db.to(bdt), None,
                dr if rdt is not None else None, None)


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
    eps = float(eps)
    if torch.is_grad_enabled() and (
            x.requires_grad or (weight is not None and weight.requires_grad) or (bias is not None and bias.requires_grad)
            or (residual is not None and residual.requires_grad)):
        return _LayerNorm.apply(x, weight, bias, eps, residual, out_dtype)
    y, s, _, _ = _forward(x, _param(weight), _param(bias), eps, residual, out_dtype, False)
    return y if residual is None else (y, s)


class LayerNorm(nn.Module):
    """Layer norm over the last dimension with a learned gain and offset (``nn.LayerNorm``'s
    parameters and state dict), through :func:`layer_norm`. ``forward(x, residual)`` adds the
    residual first and returns (y, x + residual)."""

    def __init__(self, hidden_size: int, eps: float = 1e-5, device=None, dtype=None):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(hidden_size, device=device, dtype=dtype))
        self.bias = nn.Parameter(torch.zeros(hidden_size, device=device, dtype=dtype))

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None, out_dtype: torch.dtype | None = None):
        return layer_norm(x, self.weight, self.bias, self.eps, residual, out_dtype)
