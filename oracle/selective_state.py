"""Oracle for the selective state mixer's operators (test infrastructure; see
``oracle/__init__.py``): the formulas of the published Mamba layer, step by step in float64.

Sequences are given by their offsets ``cu`` (a list); rows outside of every sequence give
zeros. ``absolute`` evaluates the same sums over absolute values: the size that rounding
errors of the result are measured against.
"""
from __future__ import annotations

import torch


def _silu(v):
    return v * torch.sigmoid(v)


def _silu_grad(v):
    s = torch.sigmoid(v)
    return s * (1 + v * (1 - s))


def _silu_grad_size(v):
    """silu' = s + v s (1 - s) is a sum too, and vanishes near v = -1.28: its terms' sizes."""
    s = torch.sigmoid(v)
    return s + v.abs() * s * (1 - s)


def conv(x, w, b, cu, silu=True, windows=None, dy=None):
    """x (rows, C), w (C, K), windows: per sequence (K - 1, C) or None. Returns a dict: y, the
    windows left behind, and with dy the gradients dx, dw, db and the absolute sums of the
    latter (aw, ab)."""
    rows, C = x.shape
    K = w.shape[1]
    out = {"y": torch.zeros_like(x), "windows": [], "dx": torch.zeros_like(x), "dw": torch.zeros_like(w),
           "db": torch.zeros(C, dtype=x.dtype), "aw": torch.zeros_like(w), "ab": torch.zeros(C, dtype=x.dtype)}
    for s in range(len(cu) - 1):
        lo, hi = cu[s], cu[s + 1]
        head = torch.zeros(K - 1, C, dtype=x.dtype) if windows is None or windows[s] is None else windows[s]
        seen = torch.cat([head, x[lo:hi]])
        out["windows"].append(seen[hi - lo:])
        if hi == lo:
            continue
        n = hi - lo
        taps = torch.stack([seen[k:k + n] for k in range(K)])  # (K, n, C)
        pre = (taps * w.t()[:, None]).sum(0) + (0 if b is None else b)
        out["y"][lo:hi] = _silu(pre) if silu else pre
        if dy is not None:
            d = dy[lo:hi] * (_silu_grad(pre) if silu else 1)
            far = torch.cat([d, torch.zeros(K - 1, C, dtype=x.dtype)])
            out["dx"][lo:hi] = sum(far[K - 1 - k:K - 1 - k + n] * w[:, k] for k in range(K))
            out["dw"] += (taps * d).sum(1).t()
            out["db"] += d.sum(0)
            out["aw"] += (taps * d).abs().sum(1).t()
            out["ab"] += d.abs().sum(0)
    return out


def scan(x, dt, A, B, C, cu, D=None, z=None, dt_bias=None, softplus=True, h0=None, dy=None, absolute=False):
    """x, dt, z (rows, C); B, C (rows, G, N); A (C, N); h0: per sequence (C, N) or None. Returns
    a dict: y, the last states h, and with dy all gradients."""
    rows, ch = x.shape
    G, N = B.shape[-2:]
    f = (lambda t: t.abs()) if absolute else (lambda t: t)
    raw = dt if dt_bias is None else dt + dt_bias
    d = torch.where(raw > 20, raw, torch.log1p(torch.exp(raw.clamp(max=20)))) if softplus else raw
    dgrad = (torch.where(raw > 20, torch.ones_like(raw), torch.sigmoid(raw)) if softplus else torch.ones_like(raw))
    Bc, Cc = (f(t).repeat_interleave(ch // G, 1) for t in (B, C))
    xf, Df = f(x), torch.zeros(ch, dtype=x.dtype) if D is None else f(D)
    zero = torch.zeros(ch, N, dtype=x.dtype)
    out = {"y": torch.zeros_like(x), "h": []}
    if dy is not None:
        out |= {"dx": torch.zeros_like(x), "ddt": torch.zeros_like(x), "dA": torch.zeros_like(A),
                "dB": torch.zeros_like(B), "dC": torch.zeros_like(C), "dD": torch.zeros(ch, dtype=x.dtype),
                "ddt_bias": torch.zeros(ch, dtype=x.dtype), "dz": torch.zeros_like(x)}
    for s in range(len(cu) - 1):
        lo, hi = cu[s], cu[s + 1]
        h = zero if h0 is None or h0[s] is None else f(h0[s])
        states, vs = [h], []
        for t in range(lo, hi):
            h = torch.exp(d[t, :, None] * A) * h + f(d[t] * x[t])[:, None] * Bc[t]
            states.append(h)
            vs.append((Cc[t] * h).sum(-1) + Df * xf[t])
            out["y"][t] = vs[-1] * (1 if z is None else f(_silu(z[t])))
        out["h"].append(h)
        if dy is None:
            continue
        carry = zero
        for t in range(hi - 1, lo - 1, -1):
            dv = f(dy[t]) if z is None else f(dy[t] * _silu(z[t]))
            if z is not None:
                out["dz"][t] = f(dy[t]) * vs[t - lo] * (_silu_grad_size if absolute else _silu_grad)(z[t])
            g = Cc[t] * dv[:, None] + carry
            a = torch.exp(d[t, :, None] * A)
            u = g * a * states[t - lo]
            gB = (g * Bc[t]).sum(-1)
            out["dB"][t] = (g * f(d[t] * x[t])[:, None]).view(G, ch // G, N).sum(1)
            out["dC"][t] = (states[t - lo + 1] * dv[:, None]).view(G, ch // G, N).sum(1)
            out["dx"][t] = f(d[t]) * gB + Df * dv
            out["ddt"][t] = ((u * f(A)).sum(-1) + xf[t] * gB) * dgrad[t]
            out["dA"] += u * f(d[t])[:, None]
            out["dD"] += dv * xf[t]
            out["ddt_bias"] += out["ddt"][t]
            carry = a * g
    return out
