"""Selective state mixer: the mixer that the pre-norm block runs for ``ssm: selective_state``.

    in_proj (C -> 2 * expand * C) -> split (u, z)
    u: causal depthwise convolution (d_conv taps) -> SiLU
    x_proj(u) -> step (dt_rank), B, C (d_state each); dt = dt_proj(step)
    y = selective scan of u with the gate silu(z) -> out_proj (expand * C -> C)

Parameter names and initial values follow the published Mamba layer (in_proj, conv1d, x_proj,
dt_proj, A_log, D, out_proj), which the reference takes from mamba_ssm for its ``mamba``
backbone (models/mamba_block.py:105-299). The projections are cuBLAS GEMMs; the convolution
and the scan read their outputs in place, at the projections' row strides.

Three forms: training and whole sequences (``forward(x)``), prompts of many lengths with a
cache (``forward(x, cu_seqlens=..., cache=..., slots=..., fresh=...)``), and one token per
sequence (``step(x, cache, slots)``; ``forward`` of one-row sequences with a cache takes it).
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch
import torch.nn.functional as F
from torch import nn

from .conv import short_conv, short_conv_step
from .scan import selective_state_scan, selective_state_step


@dataclass
class MixerCache:
    """Running sequences of one mixer: ``window`` (entries, d_conv - 1, inner) in the
    activations' type, ``state`` (entries, inner, d_state) fp32. Updated in place."""

    window: torch.Tensor
    state: torch.Tensor


class SelectiveStateMixer(nn.Module):
    """Shapes: (batch, time, in_features) -> the same, or packed (rows, in_features) with
    ``cu_seqlens``.

    Args:
        in_features: input width.
        d_state: modes per channel. Default 16.
        d_conv: taps of the convolution (1 to 8). Default 4.
        expand: inner width factor. Default 2.
        dt_rank: rank of the step projection. Default ceil(in_features / 16).
        dt_min, dt_max: range of the initial steps.
        n_groups: groups of channels that share B and C. Default 1.
    """

    def __init__(self, in_features: int, d_state: int = 16, d_conv: int = 4, expand: int = 2,
                 dt_rank: int | None = None, dt_min: float = 1e-3, dt_max: float = 0.1, n_groups: int = 1):
        super().__init__()
        inner = expand * in_features
        if inner % n_groups:
            raise ValueError(f"{inner} inner channels do not fall into {n_groups} groups")
        self.in_features, self.inner_dim, self.d_state, self.d_conv = in_features, inner, d_state, d_conv
        self.n_groups = n_groups
        self.dt_rank = dt_rank if dt_rank is not None else max(1, math.ceil(in_features / 16))
        self.in_proj = nn.Linear(in_features, 2 * inner, bias=False)
        self.conv1d = nn.Conv1d(inner, inner, kernel_size=d_conv, groups=inner, padding=d_conv - 1)
        self.x_proj = nn.Linear(inner, self.dt_rank + 2 * n_groups * d_state, bias=False)
        self.dt_proj = nn.Linear(self.dt_rank, inner, bias=True)
        self.A_log = nn.Parameter(torch.log(torch.arange(1, d_state + 1, dtype=torch.float32).repeat(inner, 1)))
        self.D = nn.Parameter(torch.ones(inner))
        self.out_proj = nn.Linear(inner, in_features, bias=False)
        with torch.no_grad():
            bound = self.dt_rank ** -0.5
            self.dt_proj.weight.uniform_(-bound, bound)
            dt = torch.exp(torch.rand(inner) * (math.log(dt_max) - math.log(dt_min)) + math.log(dt_min))
            self.dt_proj.bias.copy_(dt + torch.log(-torch.expm1(-dt)))
        self.dt_proj.bias._no_reinit = True
        self.A_log._no_weight_decay = True
        self.D._no_weight_decay = True

    def allocate_cache(self, entries: int, dtype: torch.dtype | None = None, device=None) -> MixerCache:
        """A zeroed cache of ``entries`` sequences; ``dtype``: the activations' type (that of
        the weights by default; bf16 under bf16 autocast)."""
        w = self.in_proj.weight
        dev = w.device if device is None else device
        return MixerCache(torch.zeros(entries, self.d_conv - 1, self.inner_dim, device=dev, dtype=dtype or w.dtype),
                          torch.zeros(entries, self.inner_dim, self.d_state, device=dev, dtype=torch.float32))

    def _operands(self, u):
        """(dt, B, C) of the convolved rows u."""
        N, G = self.d_state, self.n_groups
        r = self.dt_rank
        rows = self.x_proj(u)
        dt = F.linear(rows[..., :r], self.dt_proj.weight)
        B, C = (rows[..., r + i * G * N:r + (i + 1) * G * N].unflatten(-1, (G, N)) for i in range(2))
        return dt, B, C

    def forward(self, x: torch.Tensor, inference_params=None, cu_seqlens: torch.Tensor | None = None,
                cache: MixerCache | None = None, slots: torch.Tensor | None = None,
                fresh: torch.Tensor | None = None) -> torch.Tensor:
        # ``inference_params`` is accepted for the pre-norm Block's calling convention; the
        # state of running sequences is in ``cache``.
        del inference_params
        if cache is None and (slots is not None or fresh is not None):
            raise ValueError("SelectiveStateMixer: slots / fresh without a cache")
        if cache is not None and fresh is None and cu_seqlens is None and x.dim() == 3 and x.shape[1] == 1:
            return self.step(x[:, 0], cache, slots).unsqueeze(1)
        xz = self.in_proj(x)
        u, z = xz[..., :self.inner_dim], xz[..., self.inner_dim:]
        window, state = (None, None) if cache is None else (cache.window, cache.state)
        pool = {} if cache is None else {"slots": slots, "fresh": fresh}
        u = short_conv(u, self.conv1d.weight, self.conv1d.bias, cu_seqlens=cu_seqlens, state=window, **pool)
        dt, B, C = self._operands(u)
        y = selective_state_scan(u, dt, -torch.exp(self.A_log.float()), B, C, D=self.D, z=z,
                                 dt_bias=self.dt_proj.bias, cu_seqlens=cu_seqlens, state=state, **pool)
        return self.out_proj(y)

    def step(self, x: torch.Tensor, cache: MixerCache, slots: torch.Tensor | None = None) -> torch.Tensor:
        """One token per sequence, x (sequences, in_features); the cache moves on in place."""
        xz = self.in_proj(x)
        u, z = xz[..., :self.inner_dim], xz[..., self.inner_dim:]
        u = short_conv_step(u, cache.window, self.conv1d.weight, self.conv1d.bias, slots=slots)
        dt, B, C = self._operands(u)
        y = selective_state_step(u, dt, -torch.exp(self.A_log.float()), B, C, cache.state, D=self.D, z=z,
                                 dt_bias=self.dt_proj.bias, slots=slots)
        return self.out_proj(y)
