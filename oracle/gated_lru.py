"""Oracle for the gated linear recurrence (test infrastructure; see ``oracle/__init__.py``): its
formulas, step by step in float64, and its gradients by the chain rule.

Sequences are given by their offsets ``cu`` (a list); rows outside of every sequence give zeros.
``absolute`` evaluates the same sums over absolute values: the size that rounding errors of the
result are measured against.
"""
from __future__ import annotations

import torch

from .selective_state import _silu, _silu_grad, _silu_grad_size

LEAST = 1e-6  # of 1 - a^2


def parts(r, i, rate, r_bias=None, i_bias=None, scale=8.0):
    """(rho, iota, speed, a, 1 - a^2, gain) of rows r, i."""
    rho = torch.sigmoid(r if r_bias is None else r + r_bias)
    iota = torch.sigmoid(i if i_bias is None else i + i_bias)
    speed = scale * torch.where(rate > 20, rate, torch.log1p(torch.exp(rate.clamp(max=20))))
    left = -torch.expm1(-2 * speed * rho)
    return rho, iota, speed, torch.exp(-speed * rho), left, left.clamp(min=LEAST).sqrt()


def scan(x, r, i, rate, cu, z=None, r_bias=None, i_bias=None, scale=8.0, h0=None, dy=None, absolute=False):
    """x, r, i, z (rows, C); rate, r_bias, i_bias (C,); h0: per sequence (C,) or None. Returns a dict:
    y, the last states h, and with dy all gradients."""
    f = (lambda t: t.abs()) if absolute else (lambda t: t)
    rho, iota, speed, a, left, gain = parts(r, i, rate, r_bias, i_bias, scale)
    slope = scale * torch.where(rate > 20, torch.ones_like(rate), torch.sigmoid(rate))
    C = x.shape[1]
    zero = torch.zeros(C, dtype=x.dtype)
    out = {"y": torch.zeros_like(x), "h": []}
    if dy is not None:
        out |= {k: torch.zeros_like(x) for k in ("dx", "dr", "di", "dz")}
        out |= {k: zero.clone() for k in ("drate", "dr_bias", "di_bias")}
    for s in range(len(cu) - 1):
        lo, hi = cu[s], cu[s + 1]
        h = zero if h0 is None or h0[s] is None else f(h0[s])
        states = [h]
        for t in range(lo, hi):
            h = a[t] * h + gain[t] * iota[t] * f(x[t])
            states.append(h)
            out["y"][t] = h if z is None else h * f(_silu(z[t]))
        out["h"].append(h)
        if dy is None:
            continue
        carry = zero
        for t in range(hi - 1, lo - 1, -1):
            g = f(dy[t] if z is None else dy[t] * _silu(z[t])) + carry
            if z is not None:
                out["dz"][t] = f(dy[t]) * states[t - lo + 1] * (_silu_grad_size if absolute else _silu_grad)(z[t])
            through = torch.where(left[t] > LEAST, g * iota[t] * f(x[t]) * a[t] ** 2 / gain[t], zero)
            dla = g * a[t] * states[t - lo] + (through if absolute else -through)
            out["dx"][t] = g * gain[t] * iota[t]
            out["di"][t] = out["dx"][t] * f(x[t]) * (1 - iota[t])
            out["dr"][t] = (1 if absolute else -1) * speed * dla * rho[t] * (1 - rho[t])
            out["drate"] += (1 if absolute else -1) * slope * rho[t] * dla
            out["dr_bias"] += out["dr"][t]
            out["di_bias"] += out["di"][t]
            carry = a[t] * g
    return out
