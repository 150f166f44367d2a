"""Gated linear recurrence (``semx_gated_lru_fwd/bwd``, ``semx_gated_lru_step``): one real mode per
channel whose decay and input are gated per token.

    rho  = sigmoid(r + r_bias)                        iota = sigmoid(i + i_bias)
    a    = exp(-rate_scale softplus(rate) rho)        gain = sqrt(max(1 - a^2, 1e-6))
    h[t] = a[t] h[t-1] + gain[t] iota[t] x[t]         y = h silu(z)  (h without z)

* :func:`gated_lru_scan` — whole sequences: training, and prompts with a state pool.
* :func:`gated_lru_step` — one token of every sequence.
* :class:`GatedLruMixer` — the mixer that the pre-norm block runs for ``ssm: gated_lru``.

Next to :func:`~semambaxlinoss_b200.selective_state.selective_state_scan`, with which it shares the
batch (whole, packed, pooled, single tokens), a channel keeps one number instead of ``d_state``, so
a token costs a hundredth of the work and the memory's speed is the bound. The state and everything
that is summed are fp32.
"""
from __future__ import annotations

import functools
import math

import torch
import torch.nn.functional as F
from torch import nn

from . import _lib
from .selective_state._batch import TYPES, batch, check_same, rows_of, set_pool
from .selective_state.conv import short_conv, short_conv_step
from .selective_state.mixer import MixerCache


def _check(op, x, r, i, rate, z, r_bias, i_bias, rate_scale):
    """Shapes and types; returns the channels."""
    shape, dtype, dev = x.shape, x.dtype, x.get_device()
    ch = shape[-1]
    if not (rate_scale > 0 and math.isfinite(rate_scale)):
        raise ValueError(f"{op}: rate_scale must be above 0, got {rate_scale}")
    # One expression for the calls that are right, which a decoding loop makes thousands of.
    if not (r.shape == shape and i.shape == shape and r.dtype == dtype and i.dtype == dtype and r.get_device() == dev
            and i.get_device() == dev and rate.shape == (ch,) and rate.dtype in TYPES and rate.get_device() == dev
            and (z is None or (z.shape == shape and z.dtype == dtype and z.get_device() == dev))
            and (r_bias is None or (r_bias.shape == (ch,) and r_bias.dtype in TYPES and r_bias.get_device() == dev))
            and (i_bias is None or (i_bias.shape == (ch,) and i_bias.dtype in TYPES and i_bias.get_device() == dev))):
        for name, t in (("r", r), ("i", i), ("z", z)):
            if t is not None:
                check_same(op, name, t, shape, (dtype,), dev)
        for name, t in (("rate", rate), ("r_bias", r_bias), ("i_bias", i_bias)):
            if t is not None:
                check_same(op, name, t, (ch,), TYPES, dev)
    return ch


def _grads_wanted(x, r, i, rate, z, r_bias, i_bias):
    return torch.is_grad_enabled() and (
        x.requires_grad or r.requires_grad or i.requires_grad or rate.requires_grad
        or (z is not None and z.requires_grad) or (r_bias is not None and r_bias.requires_grad)
        or (i_bias is not None and i_bias.requires_grad))


def _args(x, r, i, rate, z, r_bias, i_bias, scale, S, rows, L, cu):
    """The argument struct, and what has to outlive the call. Parameters are fp32 here."""
    ch = rate.shape[0]
    x, ldx = rows_of(x, ch)
    r, ldr = rows_of(r, ch)
    i, ldi = rows_of(i, ch)
    a = _lib.new_args(_lib.SemxGatedLruArgs)
    a.bf16, a.rate_scale = x.dtype == torch.bfloat16, scale
    a.S, a.rows, a.L, a.C = S, rows, L, ch
    a.ldx, a.ldr, a.ldi = ldx, ldr, ldi
    a.x, a.r, a.i, a.rate = x.data_ptr(), r.data_ptr(), i.data_ptr(), rate.data_ptr()
    if z is not None:
        z, a.ldz = rows_of(z, ch)
        a.z = z.data_ptr()
    if r_bias is not None:
        a.r_bias = r_bias.data_ptr()
    if i_bias is not None:
        a.i_bias = i_bias.data_ptr()
    if cu is not None:
        a.cu_seqlens = cu.data_ptr()
    return a, (x, r, i, z)


@functools.lru_cache(maxsize=256)
def _sizes(S, rows, L, C, packed):
    """Bytes of the kept states, and of the workspace forward and backward: the library's, which depend
    on nothing else."""
    a = _lib.new_args(_lib.SemxGatedLruArgs)
    a.rate_scale, a.S, a.rows, a.L, a.C = 1.0, S, rows, L, C
    a.ldx = a.ldr = a.ldi = a.ldz = C
    if packed:
        a.cu_seqlens = 256
    lib = _lib.load()
    return (lib.semx_gated_lru_ckpt_bytes(a), lib.semx_gated_lru_workspace_bytes(a, 0),
            lib.semx_gated_lru_workspace_bytes(a, 1))


def _workspace(a, nbytes, like):
    if not nbytes:
        return None
    ws = _lib.scratch(nbytes, like)
    a.workspace = ws.data_ptr()
    return ws


class _GatedLru(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, r, i, rate, z, r_bias, i_bias, scale, S, rows, L, cu):
        rate32, rb32, ib32 = _lib.param32(rate), _lib.param32(r_bias), _lib.param32(i_bias)
        a, kept = _args(x, r, i, rate32, z, rb32, ib32, scale, S, rows, L, cu)
        y = x.new_empty(x.shape)
        kept_bytes, fwd, bwd = _sizes(S, rows, L, rate.shape[0], cu is not None)
        ckpt = _lib.scratch(kept_bytes, x)
        a.y, a.ckpt = y.data_ptr(), ckpt.data_ptr()
        ws = _workspace(a, fwd, x)
        _lib.call("semx_gated_lru_fwd", a, x.device)
        xr, rr, ir, zr = kept
        ctx.save_for_backward(xr, rr, ir, rate32, zr, rb32, ib32, ckpt, cu)
        ctx.cfg = (scale, S, rows, L, bwd, [None if t is None else t.dtype for t in (rate, r_bias, i_bias)])
        return y

    @staticmethod
    @_lib.once_differentiable
    def backward(ctx, dy):
        x, r, i, rate, z, r_bias, i_bias, ckpt, cu = ctx.saved_tensors
        scale, S, rows, L, nbytes, (rate_t, rb_t, ib_t) = ctx.cfg
        # Strides anew: hooks on saved tensors may have brought them back laid out otherwise.
        a, kept = _args(x, r, i, rate, z, r_bias, i_bias, scale, S, rows, L, cu)
        dy = _lib.as_rows(dy, x.dtype)
        dx, dr, di = x.new_empty(x.shape), x.new_empty(x.shape), x.new_empty(x.shape)
        dz = None if z is None else x.new_empty(x.shape)
        need = ctx.needs_input_grad
        drate = torch.empty_like(rate) if need[3] else None
        drb = torch.empty_like(r_bias) if r_bias is not None and need[5] else None
        dib = torch.empty_like(i_bias) if i_bias is not None and need[6] else None
        a.ckpt, a.dy, a.dx, a.d_r, a.d_i, a.dz = (ckpt.data_ptr(), dy.data_ptr(), dx.data_ptr(), dr.data_ptr(),
                                                  di.data_ptr(), _lib.ptr(dz))
        a.drate, a.dr_bias, a.di_bias = _lib.ptr(drate), _lib.ptr(drb), _lib.ptr(dib)
        ws = _workspace(a, nbytes, x)
        _lib.call("semx_gated_lru_bwd", a, x.device)
        return (dx, dr, di, _lib.cast(drate, rate_t), dz, _lib.cast(drb, rb_t), _lib.cast(dib, ib_t), None, None, None,
                None, None)


def gated_lru_scan(x: torch.Tensor, r: torch.Tensor, i: torch.Tensor, rate: torch.Tensor,
                   z: torch.Tensor | None = None, r_bias: torch.Tensor | None = None,
                   i_bias: torch.Tensor | None = None, rate_scale: float = 8.0,
                   cu_seqlens: torch.Tensor | None = None, state: torch.Tensor | None = None,
                   slots: torch.Tensor | None = None, fresh: torch.Tensor | None = None) -> torch.Tensor:
    """Gated recurrence over the sequences in ``x``; y has x's shape and type.

    x, r, i, z: (S, L, C), or packed (rows, C) with ``cu_seqlens`` (see
    :func:`~semambaxlinoss_b200.selective_state.short_conv` for the batch, and for state, slots
    and fresh), of one type, bf16 or fp32, at any row stride. rate, r_bias, i_bias: (C,).

    Training: gradients flow to every operand, every sequence starts from zeros; the forward keeps
    the state of every 32nd step in fp32. Prompts: ``state`` (entries, C) fp32 is read and updated
    in place; refused while a gradient is wanted."""
    op = "gated_lru_scan"
    S, rows, L = batch(op, x, cu_seqlens)
    if _lib.in_dual_level():
        _lib.refuse_tangents(op, x, r, i, rate, z, r_bias, i_bias, state)
    ch = _check(op, x, r, i, rate, z, r_bias, i_bias, rate_scale)
    if _grads_wanted(x, r, i, rate, z, r_bias, i_bias):
        if state is not None:
            raise ValueError(f"{op}: a state is for inference; the call wants gradients")
        if slots is not None or fresh is not None:
            raise ValueError(f"{op}: slots / fresh without a state")
        return _GatedLru.apply(x, r, i, rate, z, r_bias, i_bias, float(rate_scale), S, rows, L, cu_seqlens)
    rate, r_bias, i_bias = _lib.param32(rate), _lib.param32(r_bias), _lib.param32(i_bias)
    a, kept = _args(x, r, i, rate, z, r_bias, i_bias, rate_scale, S, rows, L, cu_seqlens)
    set_pool(op, a, S, x.get_device(), state, (ch,), torch.float32, slots, fresh)
    y = x.new_empty(x.shape)
    a.y = y.data_ptr()
    ws = _workspace(a, _sizes(S, rows, L, ch, cu_seqlens is not None)[1], x)
    _lib.call("semx_gated_lru_fwd", a, x.device)
    return y


def gated_lru_step(x: torch.Tensor, r: torch.Tensor, i: torch.Tensor, rate: torch.Tensor, state: torch.Tensor,
                   z: torch.Tensor | None = None, r_bias: torch.Tensor | None = None,
                   i_bias: torch.Tensor | None = None, rate_scale: float = 8.0,
                   slots: torch.Tensor | None = None) -> torch.Tensor:
    """One token of every sequence: x, r, i, z (S, C) -> y (S, C); ``state`` (entries, C) fp32 is
    updated in place. Slots as in :func:`~semambaxlinoss_b200.selective_state.short_conv`. Not
    differentiable."""
    op = "gated_lru_step"
    if not x.is_cuda:
        raise RuntimeError(f"{op} requires CUDA tensors.")
    if x.dim() != 2 or x.dtype not in TYPES:
        raise ValueError(f"{op}: x must be fp32 or bf16 (sequences, channels), got {x.dtype} {tuple(x.shape)}")
    if state is None:
        raise ValueError(f"{op}: a state is needed")
    if _lib.in_dual_level():
        _lib.refuse_tangents(op, x, r, i, rate, state, z, r_bias, i_bias)
    ch = _check(op, x, r, i, rate, z, r_bias, i_bias, rate_scale)
    if _grads_wanted(x, r, i, rate, z, r_bias, i_bias):
        raise ValueError(f"{op}: a state is for inference; the call wants gradients")
    S = x.shape[0]
    rate, r_bias, i_bias = _lib.param32(rate), _lib.param32(r_bias), _lib.param32(i_bias)
    a, kept = _args(x, r, i, rate, z, r_bias, i_bias, rate_scale, S, S, 1, None)
    set_pool(op, a, S, x.get_device(), state, (ch,), torch.float32, slots, None)
    y = x.new_empty(x.shape)
    a.y = y.data_ptr()
    _lib.call("semx_gated_lru_step", a, x.device)
    return y


class GatedLruMixer(nn.Module):
    """Mixer around the gated recurrence. Shapes: (batch, time, in_features) -> the same, or packed
    (rows, in_features) with ``cu_seqlens``.

        in_proj (C -> 2 * expand * C) -> split (u, z)
        u: causal depthwise convolution (d_conv taps)
        gate_proj(u) -> two codes of gate_rank; r = r_proj(code), i = i_proj(code)
        y = gated recurrence of u with the gate silu(z) -> out_proj (expand * C -> C)

    Args:
        in_features: input width.
        d_conv: taps of the convolution (1 to 8). Default 4.
        expand: inner width factor. Default 2.
        gate_rank: rank of the gates' projections. Default ceil(in_features / 16).
        rate_scale: scale of the decay's exponent. Default 8.
        decay_min, decay_max: range of the initial decays where the gate is open.
    """

    def __init__(self, in_features: int, d_conv: int = 4, expand: int = 2, gate_rank: int | None = None,
                 rate_scale: float = 8.0, decay_min: float = 0.9, decay_max: float = 0.999):
        super().__init__()
        if not 0 < decay_min <= decay_max < 1:
            raise ValueError(f"initial decays must lie between 0 and 1, got {decay_min} to {decay_max}")
        inner = expand * in_features
        self.in_features, self.inner_dim, self.d_conv, self.rate_scale = in_features, inner, d_conv, rate_scale
        self.gate_rank = gate_rank if gate_rank is not None else max(1, math.ceil(in_features / 16))
        self.in_proj = nn.Linear(in_features, 2 * inner, bias=False)
        self.conv1d = nn.Conv1d(inner, inner, kernel_size=d_conv, groups=inner, padding=d_conv - 1)
        self.gate_proj = nn.Linear(inner, 2 * self.gate_rank, bias=False)
        self.r_proj = nn.Linear(self.gate_rank, inner, bias=True)
        self.i_proj = nn.Linear(self.gate_rank, inner, bias=True)
        self.rate = nn.Parameter(torch.empty(inner))
        self.out_proj = nn.Linear(inner, in_features, bias=False)
        with torch.no_grad():
            # softplus(rate) rate_scale = -log(decay)
            decay = torch.rand(inner) * (decay_max - decay_min) + decay_min
            self.rate.copy_(torch.log(torch.expm1(-torch.log(decay) / rate_scale)))
        self.rate._no_weight_decay = True

    def allocate_cache(self, entries: int, dtype: torch.dtype | None = None, device=None) -> MixerCache:
        """A zeroed cache of ``entries`` sequences (``window`` (entries, d_conv - 1, inner), ``state``
        (entries, inner) fp32); ``dtype``: the activations' type (that of the weights by default;
        bf16 under bf16 autocast)."""
        w = self.in_proj.weight
        dev = w.device if device is None else device
        return MixerCache(torch.zeros(entries, self.d_conv - 1, self.inner_dim, device=dev, dtype=dtype or w.dtype),
                          torch.zeros(entries, self.inner_dim, device=dev, dtype=torch.float32))

    def _gates(self, u):
        """(r, i) of the convolved rows u, without their biases."""
        codes = self.gate_proj(u)
        return (F.linear(codes[..., :self.gate_rank], self.r_proj.weight),
                F.linear(codes[..., self.gate_rank:], self.i_proj.weight))

    def forward(self, x: torch.Tensor, inference_params=None, cu_seqlens: torch.Tensor | None = None,
                cache: MixerCache | None = None, slots: torch.Tensor | None = None,
                fresh: torch.Tensor | None = None) -> torch.Tensor:
        # ``inference_params`` is accepted for the pre-norm Block's calling convention; the
        # state of running sequences is in ``cache``.
        del inference_params
        if cache is None and (slots is not None or fresh is not None):
            raise ValueError("GatedLruMixer: slots / fresh without a cache")
        if cache is not None and fresh is None and cu_seqlens is None and x.dim() == 3 and x.shape[1] == 1:
            return self.step(x[:, 0], cache, slots).unsqueeze(1)
        xz = self.in_proj(x)
        u, z = xz[..., :self.inner_dim], xz[..., self.inner_dim:]
        window, state = (None, None) if cache is None else (cache.window, cache.state)
        pool = {} if cache is None else {"slots": slots, "fresh": fresh}
        u = short_conv(u, self.conv1d.weight, self.conv1d.bias, activation=None, cu_seqlens=cu_seqlens, state=window,
                       **pool)
        r, i = self._gates(u)
        y = gated_lru_scan(u, r, i, self.rate, z=z, r_bias=self.r_proj.bias, i_bias=self.i_proj.bias,
                           rate_scale=self.rate_scale, cu_seqlens=cu_seqlens, state=state, **pool)
        return self.out_proj(y)

    def step(self, x: torch.Tensor, cache: MixerCache, slots: torch.Tensor | None = None) -> torch.Tensor:
        """One token per sequence, x (sequences, in_features); the cache moves on in place."""
        xz = self.in_proj(x)
        u, z = xz[..., :self.inner_dim], xz[..., self.inner_dim:]
        u = short_conv_step(u, cache.window, self.conv1d.weight, self.conv1d.bias, activation=None, slots=slots)
        r, i = self._gates(u)
        y = gated_lru_step(u, r, i, self.rate, cache.state, z=z, r_bias=self.r_proj.bias, i_bias=self.i_proj.bias,
                           rate_scale=self.rate_scale, slots=slots)
        return self.out_proj(y)
