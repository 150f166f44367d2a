"""What the fp32 gated projection's sums may be off, and a model of them on the CPU.

eps = 2^-24. A product of depth K is taken in runs of 128, each 8 additions of 16 terms in the tensor cores, which
may cut where an addition rounds: 1 eps of the partial sum on average. Where terms do not cancel the k-th partial sum
is k / 8 of the run: (1 + ... + 8) / 8 = 4.5 eps; where they do, the partial sums are no larger on average.
The n = ceil(K / 128) runs are added in registers, which rounds to either side: sqrt(n) eps for the root mean
square. Left out parts and the small products' own sums: 1 eps each, and half of one more. One product:
p(K) = 7 + sqrt(n).

Root mean square errors, relative to the root mean square of the result:
* h = u act(g): u and g are p(D) off; |act'| |g| / |act| is at most 2 for silu where act counts, so 3 p(D), and 16 of
  the activation, the products and the rounding.
* du = dh act(g), dg = dh u act'(g) are no worse than 4 p(D) + 16 (act'' counts once more), their parts as above; dx
  adds p(2 H) and dw p(rows) and 2 of the store; db adds sqrt(rows) of its own, which 4 p covers below.
"""
from __future__ import annotations

import math

import torch

EPS = 2.0 ** -24


def p(depth):
    return 7 + math.sqrt(-(-depth // 128))


def allowed(name, rows, D, H):
    """Largest relative root mean square error of a result, in absolute numbers."""
    if name == "h":
        return (3 * p(D) + 16) * EPS
    return (4 * p(D) + 16 + (p(2 * H) if name == "dx" else p(rows)) + 2) * EPS


def off(got, want):
    return float((got.double().cpu() - want).norm() / want.norm())


# Random signs (what parts that are left out show in) and one sign (what sums that are cut show in): each deep in one
# of the three products.
CASES = [("random", 200, 128, 64), ("random", 300, 1000, 40), ("random", 130, 72, 1100), ("random", 3000, 40, 24),
         ("same", 40, 6000, 24), ("same", 60, 40, 3500), ("same", 24000, 24, 20)]


def inputs(signs, rows, D, H):
    """x, w, dh in fp32 values: normal, or between 0.5 and 1.5 with sums near 1."""
    g = torch.Generator().manual_seed(rows + D + H)
    if signs == "random":
        x, w, dh = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((rows, D), (2 * H, D), (rows, H)))
        return x.float(), (w * D ** -0.5).float(), dh.float()
    x, w, dh = (torch.rand(*s, generator=g, dtype=torch.float64) + 0.5 for s in ((rows, D), (2 * H, D), (rows, H)))
    return x.float(), (w / D).float(), dh.float()


def exact(x, w, dh):
    """h, dx and dw in float64, silu."""
    x, w, dh = x.double(), w.double(), dh.double()
    u, g = (x @ w.t()).chunk(2, 1)
    s = torch.sigmoid(g)
    d = torch.cat([dh * g * s, dh * u * s * (1 + g * (1 - s))], 1)
    return {"h": u * g * s, "dx": d @ w, "dw": d.t() @ x}


def cut(v):
    """float64 values cut to 24 bits towards 0."""
    return (v.view(torch.int64) & -(1 << 29)).view(torch.float64)


def parts_of(v):
    out, rest = [], v
    for _ in range(3):
        out.append(rest.to(torch.bfloat16).double())
        rest = (rest.double() - out[-1]).float()
    return out


def product(a, b, products=6, drain=128):
    """a (M, K) times b (N, K) transposed, fp32 as the kernel takes it: the first ``products`` of the parts' products
    (largest first), the first one's sums leaving the accumulator every ``drain`` of the depth (0: never)."""
    A, B = parts_of(a), parts_of(b)
    K = a.shape[1]
    order = [(0, 1), (1, 0), (1, 1), (0, 2), (2, 0)][:products - 1]
    total = small = acc = torch.zeros(a.shape[0], b.shape[0], dtype=torch.float64)
    for k in range(0, K, 16):
        s = slice(k, k + 16)
        acc = cut(acc + A[0][:, s] @ B[0][:, s].t())
        for i, j in order:
            small = cut(small + A[i][:, s] @ B[j][:, s].t())
        if drain and (k + 16) % drain == 0:
            total, acc = (total + acc).float().double(), torch.zeros_like(acc)
    return ((total + acc).float().double() + small).float()


def model(x, w, dh, **kw):
    """h, dx and dw as the kernels make them, the elementwise steps rounded to fp32."""
    H = w.shape[0] // 2
    both = product(x, w, **kw).double()
    u, g = both[:, :H], both[:, H:]
    s = torch.sigmoid(g)
    d = torch.cat([dh.double() * g * s, dh.double() * u * s * (1 + g * (1 - s))], 1).float()
    return {"h": (u * g * s).float(), "dx": product(d, w.t().contiguous(), **kw),
            "dw": product(d.t().contiguous(), x.t().contiguous(), **kw)}
