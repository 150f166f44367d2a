"""Oracle for the gated projection (test infrastructure; see ``oracle/__init__.py``): its formulas and
their gradients in float64. ``size`` of each result is the same sum over absolute values, against which
rounding errors are measured."""
from __future__ import annotations

import math

import torch


def act(g, kind):
    """(act(g), act'(g), and the size of act''s terms)."""
    if kind == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s)), s + g.abs() * s * (1 - s)
    cdf = 0.5 * torch.special.erfc(-g / math.sqrt(2))
    pdf = torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    return g * cdf, cdf + g * pdf, cdf + g.abs() * pdf


def gated(x, w, b, kind, dh=None):
    """x (rows, D), w (2 H, D), b (2 H,) or None; returns {name: (value, size)} of h and, with dh, of dx,
    dw and db."""
    H = w.shape[0] // 2
    both = x @ w.t() + (0 if b is None else b)
    size = x.abs() @ w.abs().t() + (0 if b is None else b.abs())
    u, g = both[:, :H], both[:, H:]
    su, sg = size[:, :H], size[:, H:]
    a, slope, slope_size = act(g, kind)
    # An error e of u's or g's sums reaches h as e |act(g)| or e |u act'(g)| (|act'| < 1.13).
    out = {"h": (u * a, su * a.abs() + 1.13 * u.abs() * sg + (u * a).abs())}
    if dh is None:
        return out
    d = torch.cat([dh * a, dh * u * slope], 1)
    # |act''| < 0.8: what errors of u and g do to du and dg.
    ds = torch.cat([dh.abs() * (a.abs() + 1.13 * sg), dh.abs() * (su * slope_size + 0.8 * u.abs() * sg)], 1)
    out["dx"] = (d @ w, ds @ w.abs(), d.abs() @ w.abs())
    out["dw"] = (d.t() @ x, ds.t() @ x.abs(), d.abs().t() @ x.abs())
    out["db"] = (d.sum(0), ds.sum(0), d.abs().sum(0))
    return out
