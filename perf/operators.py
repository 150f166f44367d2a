"""Timing cases of the selective state mixer's operators and of the layer norm.

Four kinds of pass ("op" of a case):

* ``conv``  the short causal convolution with its SiLU over whole sequences;
* ``scan``  the selective state scan over whole sequences;
* ``step``  one token of every running sequence: the convolution's single-token form, then the
  scan's (between them the model has its own products, so the scan's operands are inputs here);
* ``norm``  the layer norm, alone or with the residual added first.

``conv`` and ``scan`` come as a prompt (``train`` false: the sequences start from and leave their
state in a pool) and as training (``train`` true: outputs and all gradients). ``ragged`` says
whether the sequences are packed one behind the other, with some unused rows at the end, or have
one length. With ``own`` false a pass runs the plain form below, elementary torch operations in
32 bits; with ``own`` true it calls the package.
"""
import math

import torch

own = False


# -- cases ------------------------------------------------------------------------------------


def listed():
    return [
        # A serving batch's prompts of many lengths: x is half of the in_proj output's rows.
        {"name": "conv prompts ragged bf16", "op": "conv", "train": False, "ragged": True, "rows": 6151, "seqs": 13,
         "width": 2048, "taps": 4, "dtype": "bf16"},
        # The frequency-axis sequences of a time-frequency block in training.
        {"name": "conv training fp32", "op": "conv", "train": True, "ragged": False, "rows": 404 * 321, "seqs": 404,
         "width": 256, "taps": 4, "dtype": "fp32"},
        # One long prompt alone: nothing but its length to spread over the GPU.
        {"name": "scan one long prompt bf16", "op": "scan", "train": False, "ragged": False, "rows": 8191, "seqs": 1,
         "width": 2048, "modes": 16, "groups": 1, "dtype": "bf16"},
        # A serving batch's prompts of many lengths.
        {"name": "scan prompts ragged bf16", "op": "scan", "train": False, "ragged": True, "rows": 4099, "seqs": 24,
         "width": 4096, "modes": 16, "groups": 1, "dtype": "bf16"},
        # Three short utterances of a small model: latency.
        {"name": "scan short prompts fp32", "op": "scan", "train": False, "ragged": True, "rows": 150, "seqs": 3,
         "width": 256, "modes": 16, "groups": 1, "dtype": "fp32"},
        # The frequency-axis sequences of a time-frequency block in training.
        {"name": "scan training 404x321 fp32", "op": "scan", "train": True, "ragged": False, "rows": 404 * 321,
         "seqs": 404, "width": 256, "modes": 16, "groups": 1, "dtype": "fp32"},
        # A sequence model's training batch: few long sequences, many channels.
        {"name": "scan training 4x2047 bf16", "op": "scan", "train": True, "ragged": False, "rows": 4 * 2047,
         "seqs": 4, "width": 2048, "modes": 16, "groups": 1, "dtype": "bf16"},
        # One stream, frame by frame: latency.
        {"name": "step 1 row bf16", "op": "step", "seqs": 1, "width": 2048, "modes": 16, "groups": 1, "taps": 4,
         "dtype": "bf16"},
        # A full decoding batch.
        {"name": "step 192 rows bf16", "op": "step", "seqs": 192, "width": 4096, "modes": 16, "groups": 1, "taps": 4,
         "dtype": "bf16"},
        # The norm in front of a decoded token's mixer, residual added first: latency.
        {"name": "norm 7 rows bf16", "op": "norm", "train": False, "residual": True, "rows": 7, "width": 2048,
         "dtype": "bf16"},
        # The generator's training step: narrow rows, very many.
        {"name": "norm training 513600x64 fp32", "op": "norm", "train": True, "residual": False, "rows": 513600,
         "width": 64, "dtype": "fp32"},
        # A sequence model's training batch, residual stream in fp32.
        {"name": "norm training 8192x4096 bf16", "op": "norm", "train": True, "residual": True, "rows": 8192,
         "width": 4096, "dtype": "bf16"},
    ]


def _between(rng, lo, hi):
    """A whole number of [lo, hi], its logarithm spread evenly."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, hi):
    """Mostly multiples of 32 (what models have), one in four any number."""
    c = _between(rng, 48, hi)
    return c if rng.random() < 0.25 else max(64, c // 32 * 32)


def draw(rng):
    op = rng.choice(["conv", "scan", "scan", "step", "norm"])
    dtype = rng.choice(["bf16", "fp32"])
    if op == "norm":
        width = _width(rng, 8192)
        rows = _between(rng, 1, max(2, 32_000_000 // width))
        return {"op": op, "train": rng.random() < 0.5, "residual": rng.random() < 0.5, "rows": rows, "width": width,
                "dtype": dtype}
    groups = rng.choice([1, 1, 1, 2])
    if op == "step":
        width = _width(rng, 4096) // groups * groups
        return {"op": op, "seqs": _between(rng, 1, 192), "width": width, "modes": rng.choice([8, 16, 16, 16, 24]),
                "groups": groups, "taps": rng.choice([2, 3, 4, 4]), "dtype": dtype}
    width = _width(rng, 4096) // groups * groups
    train = rng.random() < 0.5
    most = (30_000_000 if op == "conv" else 14_000_000) // width
    rows = _between(rng, 64, min(max(65, most), 65536 if op == "conv" else 16384))
    seqs = min(_between(rng, 1, 400), max(1, rows // 2))
    ragged = rng.random() < 0.5
    if not ragged:
        rows = max(1, rows // seqs) * seqs
    case = {"op": op, "train": train, "ragged": ragged, "rows": rows, "seqs": seqs, "width": width, "dtype": dtype}
    if op == "conv":
        return dict(case, taps=rng.choice([2, 3, 4, 4]))
    return dict(case, modes=rng.choice([8, 16, 16, 16]), groups=groups)


_TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# -- inputs -----------------------------------------------------------------------------------


def _lengths(case, g):
    """(S + 1) row offsets: lengths from one row up, with a few unused rows behind the last."""
    S, rows = case["seqs"], case["rows"]
    if not case["ragged"]:
        return torch.arange(S + 1, dtype=torch.int64) * (rows // S)
    used = max(S, rows - min(rows // 16, 5))
    share = torch.rand(S, generator=g, dtype=torch.float64) ** 2 + 1e-3
    extra = torch.floor(share / share.sum() * (used - S)).to(torch.int64)
    return torch.cat([torch.zeros(1, dtype=torch.int64), torch.cumsum(extra + 1, 0)])


def _pool(case, S, g):
    """Slots of the sequences in a pool somewhat larger than the batch, and which are new."""
    slots = torch.randperm(S + 3, generator=g)[:S].to(torch.int32)
    fresh = torch.rand(S, generator=g) < 0.5
    return S + 3, slots.cuda(), fresh.cuda()


def prepare(case, seed):
    host = torch.Generator().manual_seed(seed)
    gpu = torch.Generator(device="cuda").manual_seed(seed)
    t = _TYPES[case["dtype"]]
    C, op = case["width"], case["op"]

    def rand(*shape, dtype=t, scale=1.0):
        return (torch.randn(*shape, generator=gpu, device="cuda") * scale).to(dtype)

    st = {"case": dict(case)}
    if op == "norm":
        n = case["rows"]
        st["x"] = rand(n, C) + 0.25
        st["weight"] = rand(C, dtype=torch.float32, scale=0.2) + 1.0
        st["bias"] = rand(C, dtype=torch.float32, scale=0.2)
        if case["residual"]:
            st["residual"] = rand(n, C, dtype=torch.float32, scale=2.0)
        if case["train"]:
            st["dy"] = rand(n, C)
            if case["residual"]:
                st["ds"] = rand(n, C, dtype=torch.float32)
        return st
    S = case["seqs"]
    if op == "step":
        lead, prompt = (S,), True
    else:
        cu = _lengths(case, host)
        st["host_cu"], st["offsets"] = cu.tolist(), cu.cuda()
        st["cu"] = cu.to(torch.int32).cuda() if case["ragged"] else None
        lead = (case["rows"],) if case["ragged"] else (S, case["rows"] // S)
        prompt = not case["train"]
    if prompt:
        n_slots, st["slots"], st["fresh"] = _pool(case, S, host)
    xz = rand(*lead, 2 * C)
    st["x"], z = xz[..., :C], xz[..., C:]
    if op in ("conv", "step"):
        K = case["taps"]
        st["conv_weight"] = rand(C, K, dtype=torch.float32, scale=K ** -0.5)
        st["conv_bias"] = rand(C, dtype=torch.float32, scale=0.1)
        if prompt:
            st["window"] = rand(n_slots, K - 1, C)
    if op in ("scan", "step"):
        N, G = case["modes"], case["groups"]
        st["z"] = z
        if op == "step":
            st["u"] = rand(*lead, C)  # the scan's input
        st["dt"] = rand(*lead, C, scale=0.5)
        rank = max(1, C // 16)
        dbc = rand(*lead, rank + 2 * G * N)  # the rows of the token projection: step, B, C
        st["B"] = dbc[..., rank:rank + G * N].unflatten(-1, (G, N))
        st["C"] = dbc[..., rank + G * N:].unflatten(-1, (G, N))
        dt0 = torch.exp(torch.rand(C, generator=gpu, device="cuda") * math.log(100.0) + math.log(1e-3))
        st["dt_bias"] = dt0 + torch.log(-torch.expm1(-dt0))
        decay = torch.arange(1, N + 1, device="cuda", dtype=torch.float32).expand(C, N)
        st["A"] = -decay * torch.exp(rand(C, N, dtype=torch.float32, scale=0.1))
        st["D"] = rand(C, dtype=torch.float32, scale=0.5) + 1.0
        if prompt:
            st["state"] = rand(n_slots, C, N, dtype=torch.float32)
    if op != "step" and case["train"]:
        st["dy"] = rand(*lead, C)
    return st


# -- the plain forms --------------------------------------------------------------------------


def _silu(v):
    return v / (1 + torch.exp(-v))


def _silu_grad(v):
    s = 1 / (1 + torch.exp(-v))
    return s * (1 + v * (1 - s))


def _softplus(v):
    return torch.where(v > 20, v, torch.log1p(torch.exp(torch.clamp(v, max=20))))


def _rows_of(st):
    """Per row: the position in its sequence, the sequence, and whether it belongs to one."""
    rows, cu = st["case"]["rows"], st["offsets"]
    at = torch.arange(rows, device="cuda")
    seq = torch.searchsorted(cu[1:], at, right=True)
    live = seq < cu.numel() - 1
    seq = torch.clamp(seq, max=cu.numel() - 2)
    return at - cu[seq], seq, live


def _taps(x, window, pos, seq, K):
    """(rows, K, C): the inputs that each row's convolution sees. ``window`` (S, K - 1, C): the inputs
    in front of each sequence's first row."""
    rows, tap = x.shape[0], torch.arange(K, device=x.device) - (K - 1)
    at = torch.arange(rows, device=x.device)[:, None] + tap
    back = pos[:, None] + tap  # position in the sequence; below 0: in the window
    at = torch.where(back >= 0, at, rows + seq[:, None] * (K - 1) + torch.clamp(back + K - 1, max=max(K - 2, 0)))
    return torch.cat([x, window.reshape(-1, x.shape[1])])[at]


def _conv(st):
    case = st["case"]
    C, K = case["width"], case["taps"]
    pos, seq, live = _rows_of(st)
    x = st["x"].reshape(-1, C).float()
    w, bias = st["conv_weight"], st["conv_bias"]
    on = live[:, None].float()
    if not case["train"]:
        slots = st["slots"].long()
        old = st["window"][slots].float()
        old[st["fresh"]] = 0
        seen = _taps(x, old, pos, seq, K)
        y = _silu(bias + (seen * w.t()).sum(1)) * on
        # The window left behind: the last K - 1 inputs of the sequence's old window and rows.
        cu = st["offsets"]
        length = (cu[1:] - cu[:-1])[:, None]
        back = length - (K - 1) + torch.arange(K - 1, device="cuda")
        new = x[torch.clamp(cu[:-1, None] + back, min=0, max=x.shape[0] - 1)]
        kept = torch.gather(old, 1, torch.clamp(back + K - 1, min=0, max=K - 2)[..., None].expand(-1, -1, C))
        st["window"][slots] = torch.where((back >= 0)[..., None], new, kept).to(st["window"].dtype)
        return {"y": y.to(st["x"].dtype).view(st["x"].shape), "window": st["window"]}
    seen = _taps(x, x.new_zeros(case["seqs"], K - 1, C), pos, seq, K)
    pre = bias + (seen * w.t()).sum(1)
    dpre = st["dy"].reshape(-1, C).float() * _silu_grad(pre) * on
    dw = (seen.double() * dpre[:, None].double()).sum(0).t()
    # Row t is tap k of row t + K - 1 - k of the same sequence.
    cu = st["offsets"]
    left = (cu[seq + 1] - cu[seq] - 1 - pos)[:, None]  # rows behind this one in the sequence
    ahead = K - 1 - torch.arange(K, device="cuda")
    at = torch.arange(x.shape[0], device="cuda")[:, None] + ahead
    reach = torch.where((ahead <= left)[..., None], dpre[torch.clamp(at, max=x.shape[0] - 1)],
                        torch.zeros((), device="cuda"))
    dx = (reach * w.t()).sum(1) * on
    t, shape = st["x"].dtype, st["x"].shape
    return {"y": (_silu(pre) * on).to(t).view(shape), "dx": dx.to(t).view(shape), "dw": dw.float(),
            "db": dpre.double().sum(0).float()}


def _running(a, b):
    """All h_t = a_t h_{t-1} + b_t along dim 0, from h = 0, by doubling: after the pass with distance d
    every row holds the sum over the 2 d rows up to it."""
    a, d = a.clone(), 1
    while d < a.shape[0]:
        b = torch.cat([b[:d], b[d:] + a[d:] * b[:-d]])
        a = torch.cat([a[:d], a[d:] * a[:-d]])
        d *= 2
    return b


def _per_channel(v, C, N):
    """(rows, groups, N) -> (rows, C, N): the group's values for each of its channels."""
    return v.float().reshape(-1, v.shape[-2], N).repeat_interleave(C // v.shape[-2], dim=1)


def _scan(st):
    case = st["case"]
    C, N, G = case["width"], case["modes"], case["groups"]
    pos, seq, live = _rows_of(st)
    t, shape = st["x"].dtype, st["x"].shape
    x, raw = st["x"].reshape(-1, C).float(), st["dt"].reshape(-1, C).float() + st["dt_bias"]
    z = st["z"].reshape(-1, C).float()
    Bc, Cc = _per_channel(st["B"], C, N), _per_channel(st["C"], C, N)
    step = _softplus(raw)
    a = torch.exp(step[..., None] * st["A"])
    b = (step * x)[..., None] * Bc
    first = (pos == 0)[:, None, None]
    if not case["train"]:
        slots = st["slots"].long()
        old = st["state"][slots].clone()
        old[st["fresh"]] = 0
        starts = st["offsets"][:-1]
        b[starts] += a[starts] * old
    a = torch.where(first, torch.zeros((), device="cuda"), a)
    h = _running(a, b)
    ypre = (Cc * h).sum(-1) + st["D"] * x
    on = live[:, None].float()
    y = (ypre * _silu(z) * on).to(t).view(shape)
    if not case["train"]:
        st["state"][slots] = h[st["offsets"][1:] - 1]
        return {"y": y, "state": st["state"]}
    do = st["dy"].reshape(-1, C).float() * on
    dz = do * ypre * _silu_grad(z)
    dyp = do * _silu(z)
    # g_t = C_t dy_t + a_{t+1} g_{t+1}: the running sum of the rows turned round.
    nxt = torch.cat([a[1:], torch.zeros_like(a[:1])])
    g = torch.flip(_running(torch.flip(nxt, [0]), torch.flip(Cc * dyp[..., None], [0])), [0])
    u = g * (h - b)
    gB = (g * Bc).sum(-1)
    dstep = (u * st["A"]).sum(-1) + x * gB
    ddt = dstep * torch.where(raw > 20, torch.ones((), device="cuda"), 1 / (1 + torch.exp(-raw))) * on
    rows = x.shape[0]
    dB = (g * (step * x)[..., None]).view(rows, G, C // G, N).sum(2) * on[..., None]
    dC = (h * dyp[..., None]).view(rows, G, C // G, N).sum(2)
    dx = (step * gB + st["D"] * dyp) * on
    return {"y": y, "dx": dx.to(t).view(shape), "ddt": ddt.to(t).view(shape), "dz": dz.to(t).view(shape),
            "dB": dB.to(t).view(st["B"].shape), "dC": dC.to(t).view(st["C"].shape),
            "dA": (u.double() * step[..., None].double()).sum(0).float(), "dD": (dyp.double() * x).sum(0).float(),
            "ddt_bias": ddt.double().sum(0).float()}


def _step(st):
    case = st["case"]
    C, N = case["width"], case["modes"]
    slots, t = st["slots"].long(), st["x"].dtype
    seen = torch.cat([st["window"][slots], st["x"][:, None]], 1)
    st["window"][slots] = seen[:, 1:]
    conv = _silu(st["conv_bias"] + (seen.float() * st["conv_weight"].t()).sum(1))
    x = st["u"].float()
    step = _softplus(st["dt"].float() + st["dt_bias"])
    h = torch.exp(step[..., None] * st["A"]) * st["state"][slots] + (step * x)[..., None] * _per_channel(st["B"], C, N)
    st["state"][slots] = h
    y = ((h * _per_channel(st["C"], C, N)).sum(-1) + st["D"] * x) * _silu(st["z"].float())
    return {"conv": conv.to(t), "y": y.to(t), "window": st["window"], "state": st["state"]}


_EPS = 1e-5


def _norm(st):
    case = st["case"]
    t = st["x"].dtype
    s = st["x"].float() + (st["residual"] if case["residual"] else 0)
    mean = s.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(((s - mean) * (s - mean)).mean(-1, keepdim=True) + _EPS)
    xhat = (s - mean) * rstd
    out = {"y": (xhat * st["weight"] + st["bias"]).to(t)}
    if case["residual"]:
        out["sum"] = s
    if not case["train"]:
        return out
    dy = st["dy"].float()
    gw = dy * st["weight"]
    ds = rstd * (gw - gw.mean(-1, keepdim=True) - xhat * (gw * xhat).mean(-1, keepdim=True))
    if case["residual"]:
        ds = ds + st["ds"]
        out["dresidual"] = ds
    out["dx"] = ds.to(t)
    out["dweight"] = (dy.double() * xhat).sum(0).float()
    out["dbias"] = dy.double().sum(0).float()
    return out


# -- the package's calls ----------------------------------------------------------------------


def _leaf(v):
    return v.detach().requires_grad_()


def _own_conv(st):
    from semambaxlinoss_b200.selective_state import short_conv

    case = st["case"]
    if not case["train"]:
        y = short_conv(st["x"], st["conv_weight"], st["conv_bias"], cu_seqlens=st["cu"], state=st["window"],
                       slots=st["slots"], fresh=st["fresh"])
        return {"y": y, "window": st["window"]}
    x, w, b = (_leaf(st[k]) for k in ("x", "conv_weight", "conv_bias"))
    y = short_conv(x, w, b, cu_seqlens=st["cu"])
    dx, dw, db = torch.autograd.grad(y, (x, w, b), st["dy"])
    return {"y": y, "dx": dx, "dw": dw, "db": db}


def _own_scan(st):
    from semambaxlinoss_b200.selective_state import selective_state_scan

    case = st["case"]
    if not case["train"]:
        y = selective_state_scan(st["x"], st["dt"], st["A"], st["B"], st["C"], D=st["D"], z=st["z"],
                                 dt_bias=st["dt_bias"], cu_seqlens=st["cu"], state=st["state"], slots=st["slots"],
                                 fresh=st["fresh"])
        return {"y": y, "state": st["state"]}
    names = ("x", "dt", "A", "B", "C", "D", "z", "dt_bias")
    v = {k: _leaf(st[k]) for k in names}
    y = selective_state_scan(v["x"], v["dt"], v["A"], v["B"], v["C"], D=v["D"], z=v["z"], dt_bias=v["dt_bias"],
                             cu_seqlens=st["cu"])
    grads = torch.autograd.grad(y, [v[k] for k in names], st["dy"])
    return dict({"d" + k: g for k, g in zip(names, grads)}, y=y)


def _own_step(st):
    from semambaxlinoss_b200.selective_state import selective_state_step, short_conv_step

    conv = short_conv_step(st["x"], st["window"], st["conv_weight"], st["conv_bias"], slots=st["slots"])
    y = selective_state_step(st["u"], st["dt"], st["A"], st["B"], st["C"], st["state"], D=st["D"], z=st["z"],
                             dt_bias=st["dt_bias"], slots=st["slots"])
    return {"conv": conv, "y": y, "window": st["window"], "state": st["state"]}


def _own_norm(st):
    from semambaxlinoss_b200.layer_norm import layer_norm

    case = st["case"]
    if not case["train"]:
        got = layer_norm(st["x"], st["weight"], st["bias"], eps=_EPS, residual=st.get("residual"))
        return {"y": got[0], "sum": got[1]} if case["residual"] else {"y": got}
    x, w, b = (_leaf(st[k]) for k in ("x", "weight", "bias"))
    if not case["residual"]:
        y = layer_norm(x, w, b, eps=_EPS)
        dx, dw, db = torch.autograd.grad(y, (x, w, b), st["dy"])
        return {"y": y, "dx": dx, "dweight": dw, "dbias": db}
    r = _leaf(st["residual"])
    y, s = layer_norm(x, w, b, eps=_EPS, residual=r)
    dx, dr, dw, db = torch.autograd.grad((y, s), (x, r, w, b), (st["dy"], st["ds"]))
    return {"y": y, "sum": s, "dx": dx, "dresidual": dr, "dweight": dw, "dbias": db}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"conv": _own_conv, "scan": _own_scan, "step": _own_step, "norm": _own_norm}[op](state)
    return {"conv": _conv, "scan": _scan, "step": _step, "norm": _norm}[op](state)


# -- what a pass cannot do without ------------------------------------------------------------


def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    C, op = case["width"], case["op"]
    if op == "norm":
        n = case["rows"] * C
        forward = 2 * e + (8 if case["residual"] else 0)  # x, y; residual, sum
        back = 2 * e + (8 if case["residual"] else 0)  # dy, dx; ds, dresidual
        return {"bytes": n * (forward + (back if case["train"] else 0)) + 16 * C,
                "flops": n * (20 if case["train"] else 8)}
    S = case["seqs"]
    if op == "step":
        K, N, G = case["taps"], case["modes"], case["groups"]
        per_row = 6 * C * e + 2 * (K - 1) * C * e + 8 * C * N + 2 * G * N * e
        return {"bytes": S * per_row + 4 * C * (N + K + 3), "flops": S * C * (2 * K + 7 * N + 12)}
    n = case["rows"] * C
    if op == "conv":
        K = case["taps"]
        if case["train"]:
            return {"bytes": n * 4 * e + 8 * C * (K + 1), "flops": n * (8 * K + 12)}
        return {"bytes": n * 2 * e + 2 * S * (K - 1) * C * e + 4 * C * (K + 1), "flops": n * (2 * K + 5)}
    N, G = case["modes"], case["groups"]
    if case["train"]:
        return {"bytes": n * 8 * e + 4 * case["rows"] * G * N * e + 8 * C * (N + 2), "flops": n * (24 * N + 30)}
    return {"bytes": n * 4 * e + 2 * case["rows"] * G * N * e + 8 * S * C * N + 4 * C * (N + 2),
            "flops": n * (7 * N + 12)}


# -- the definitions in 64 bits ---------------------------------------------------------------


def _padded(v, cu, width):
    """(S, longest, width) in 64 bits of the packed or equal-length rows."""
    rows = v.double().reshape(-1, width)
    longest = max(max(q - p for p, q in zip(cu[:-1], cu[1:])), 1)
    out = rows.new_zeros(len(cu) - 1, longest, width)
    for s, (p, q) in enumerate(zip(cu[:-1], cu[1:])):
        out[s, :q - p] = rows[p:q]
    return out


def _packed(v, cu, like, width):
    """The rows of a padded tensor back in their places, zeros where no sequence is."""
    rows = v.new_zeros(like.numel() // width, width)
    for s, (p, q) in enumerate(zip(cu[:-1], cu[1:])):
        rows[p:q] = v[s, :q - p].reshape(q - p, width)
    return rows.view(like.shape)


def _exact_conv(case, st):
    C, K, cu = case["width"], case["taps"], st["host_cu"]
    x = _padded(st["x"], cu, C)
    S, L, _ = x.shape
    head = x.new_zeros(S, K - 1, C)
    if not case["train"]:
        head = torch.where(st["fresh"][:, None, None], head, st["window"].double()[st["slots"].long()])
    long = torch.cat([head, x], 1)
    w = st["conv_weight"].double()
    pre = st["conv_bias"].double() + sum(long[:, k:k + L] * w[:, k] for k in range(K))
    sig = torch.sigmoid(pre)
    out = {"y": _packed(pre * sig, cu, st["x"], C)}
    if not case["train"]:
        window = st["window"].double()
        for s in range(S):
            n = cu[s + 1] - cu[s]
            window[int(st["slots"][s])] = long[s, n:n + K - 1]
        return dict(out, window=window)
    d = _padded(st["dy"], cu, C) * (sig + pre * sig * (1 - sig))
    for s in range(S):
        d[s, cu[s + 1] - cu[s]:] = 0
    far = torch.cat([d, d.new_zeros(S, K - 1, C)], 1)
    dx = sum(far[:, K - 1 - k:K - 1 - k + L] * w[:, k] for k in range(K))
    dw = torch.stack([(long[:, k:k + L] * d).sum((0, 1)) for k in range(K)], 1)
    return dict(out, dx=_packed(dx, cu, st["x"], C), dw=dw, db=d.sum((0, 1)))


def _exact_scan(case, st):
    C, N, G, cu = case["width"], case["modes"], case["groups"], st["host_cu"]
    x, z = _padded(st["x"], cu, C), _padded(st["z"], cu, C)
    raw = _padded(st["dt"], cu, C) + st["dt_bias"].double()
    S, L, _ = x.shape
    Bm, Cm = (_padded(st[k], cu, G * N).view(S, L, G, 1, N) for k in ("B", "C"))
    step = torch.nn.functional.softplus(raw)
    A, D = st["A"].double().view(G, C // G, N), st["D"].double()
    length = torch.tensor([q - p for p, q in zip(cu[:-1], cu[1:])], device=x.device)
    h = x.new_zeros(S, G, C // G, N)
    if not case["train"]:
        old = st["state"].double()[st["slots"].long()].view(h.shape)
        h = torch.where(st["fresh"][:, None, None, None], h, old)
    # What every step leaves is kept for the adjoint, 16 bytes a mode; past 24 GB there is no time for it.
    if case["train"] and S * L * C * N * 8 > 24e9:
        return None
    kept, ypre = [], torch.empty_like(x)
    for t in range(L):
        s4 = step[:, t].view(S, G, C // G, 1)
        nxt = torch.exp(s4 * A) * h + s4 * x[:, t].view(s4.shape) * Bm[:, t]
        h = nxt if case["train"] else torch.where((t < length)[:, None, None, None], nxt, h)
        if case["train"]:
            kept.append(h)
        ypre[:, t] = (h * Cm[:, t]).sum(-1).view(S, C) + D * x[:, t]
    sig = torch.sigmoid(z)
    out = {"y": _packed(ypre * z * sig, cu, st["x"], C)}
    if not case["train"]:
        state = st["state"].double()
        state[st["slots"].long()] = h.view(S, C, N)
        return dict(out, state=state)
    do = _padded(st["dy"], cu, C)
    dyp = do * z * sig
    dz = do * ypre * (sig + z * sig * (1 - sig))
    dx, ddt = torch.empty_like(x), torch.empty_like(x)
    dB, dC = torch.zeros(S, L, G, N, device=x.device, dtype=x.dtype), torch.zeros(S, L, G, N, device=x.device, dtype=x.dtype)
    dA, carry = torch.zeros_like(A), torch.zeros_like(h)
    for t in range(L - 1, -1, -1):
        s4, x4, d4 = (v[:, t].view(S, G, C // G, 1) for v in (step, x, dyp))
        g = carry + Cm[:, t] * d4
        a = torch.exp(s4 * A)
        prev = kept[t - 1] if t else torch.zeros_like(h)
        through = g * a * prev
        dC[:, t], dB[:, t] = (kept[t] * d4).sum(2), (g * s4 * x4).sum(2)
        gB = (g * Bm[:, t]).sum(-1).view(S, C)
        dx[:, t] = step[:, t] * gB + D * dyp[:, t]
        ddt[:, t] = ((through * A).sum(-1).view(S, C) + x[:, t] * gB) * torch.sigmoid(raw[:, t])
        dA += (through * s4).sum(0)
        carry = a * g
        kept.pop()
    on = (torch.arange(L, device=x.device) < length[:, None])[..., None]
    return dict(out, dx=_packed(dx, cu, st["x"], C), ddt=_packed(ddt, cu, st["x"], C), dz=_packed(dz, cu, st["x"], C),
                dB=_packed(dB, cu, st["B"], G * N), dC=_packed(dC, cu, st["C"], G * N), dA=dA.reshape(C, N),
                dD=(dyp * x).sum((0, 1)), ddt_bias=(ddt * on).sum((0, 1)))


def _exact_step(case, st):
    C, N, G, K = case["width"], case["modes"], case["groups"], case["taps"]
    slots, S = st["slots"].long(), case["seqs"]
    window, state = st["window"].double(), st["state"].double()
    seen = torch.cat([window[slots], st["x"].double()[:, None]], 1)
    window[slots] = seen[:, 1:]
    pre = st["conv_bias"].double() + torch.einsum("skc,ck->sc", seen, st["conv_weight"].double())
    x = st["u"].double()
    step = torch.nn.functional.softplus(st["dt"].double() + st["dt_bias"].double())
    Bm, Cm = (st[k].double().view(S, G, 1, N).expand(S, G, C // G, N).reshape(S, C, N) for k in ("B", "C"))
    h = torch.exp(step[..., None] * st["A"].double()) * state[slots] + (step * x)[..., None] * Bm
    state[slots] = h
    y = ((h * Cm).sum(-1) + st["D"].double() * x) * torch.nn.functional.silu(st["z"].double())
    return {"conv": pre * torch.sigmoid(pre), "y": y, "window": window, "state": state}


def _exact_norm(case, st):
    s = st["x"].double()
    if case["residual"]:
        s = s + st["residual"].double()
    var, mean = torch.var_mean(s, -1, correction=0, keepdim=True)
    xhat = (s - mean) / torch.sqrt(var + _EPS)
    w = st["weight"].double()
    out = {"y": xhat * w + st["bias"].double()}
    if case["residual"]:
        out["sum"] = s
    if not case["train"]:
        return out
    dy = st["dy"].double()
    d = case["width"]
    gw = dy * w
    ds = (gw - (gw.sum(-1, keepdim=True) + xhat * (gw * xhat).sum(-1, keepdim=True)) / d) / torch.sqrt(var + _EPS)
    if case["residual"]:
        ds = ds + st["ds"].double()
        out["dresidual"] = ds
    return dict(out, dx=ds, dweight=(dy * xhat).sum(0), dbias=dy.sum(0))


def exact(case, seed):
    st = prepare(case, seed)
    return {"conv": _exact_conv, "scan": _exact_scan, "step": _exact_step, "norm": _exact_norm}[case["op"]](case, st)
