"""Timing cases of the gated recurrence's operators and of the gated projection.

Three kinds of pass ("op" of a case):

* ``scan``  the gated linear recurrence over whole sequences, as a prompt (``train`` false: the
  sequences start from and leave their state in a pool) or as training (``train`` true: output and
  all gradients). ``ragged`` says whether the sequences are packed one behind the other, with some
  unused rows at the end, or have one length;
* ``step``  one token of every running sequence through the recurrence;
* ``mlp``   the gated projection of a feed-forward block (both projections, the activation and their
  product), forward (``train`` false) or with all gradients.

With ``own`` false a pass runs the plain form below, elementary torch operations in 32 bits; with
``own`` true it calls the package.
"""
import math

import torch

own = False


# -- cases ------------------------------------------------------------------------------------


def listed():
    return [
        # One long prompt alone: nothing but its length to spread over the GPU.
        {"name": "scan one long prompt bf16", "op": "scan", "train": False, "ragged": False, "rows": 8191, "seqs": 1,
         "width": 2048, "dtype": "bf16"},
        # A serving batch's prompts of many lengths.
        {"name": "scan prompts ragged bf16", "op": "scan", "train": False, "ragged": True, "rows": 4099, "seqs": 24,
         "width": 4096, "dtype": "bf16"},
        # Three short utterances of a small model: latency.
        {"name": "scan short prompts fp32", "op": "scan", "train": False, "ragged": True, "rows": 150, "seqs": 3,
         "width": 256, "dtype": "fp32"},
        # The frequency-axis sequences of a time-frequency block in training.
        {"name": "scan training 404x321 fp32", "op": "scan", "train": True, "ragged": False, "rows": 404 * 321,
         "seqs": 404, "width": 256, "dtype": "fp32"},
        # A sequence model's training batch: few long sequences, many channels.
        {"name": "scan training 4x2047 bf16", "op": "scan", "train": True, "ragged": False, "rows": 4 * 2047,
         "seqs": 4, "width": 2048, "dtype": "bf16"},
        # One stream, frame by frame: latency.
        {"name": "step 1 row bf16", "op": "step", "seqs": 1, "width": 2048, "dtype": "bf16"},
        # A full decoding batch.
        {"name": "step 192 rows fp32", "op": "step", "seqs": 192, "width": 4096, "dtype": "fp32"},
        # The feed-forward half of a block for one decoded token: the weights' bytes.
        {"name": "mlp 1 row bf16", "op": "mlp", "train": False, "rows": 1, "width": 2048, "hidden": 5504,
         "act": "silu", "bias": False, "dtype": "bf16"},
        # A full decoding batch: the weights' bytes and a part of a tile of rows.
        {"name": "mlp 192 rows bf16", "op": "mlp", "train": False, "rows": 192, "width": 4096, "hidden": 11008,
         "act": "silu", "bias": False, "dtype": "bf16"},
        # A serving batch's prompts; the hidden width is 8/3 of the width, not rounded.
        {"name": "mlp prompts odd bf16", "op": "mlp", "train": False, "rows": 4099, "width": 2048, "hidden": 5461,
         "act": "gelu", "bias": True, "dtype": "bf16"},
        # A sequence model's training batch.
        {"name": "mlp training 8192x2048 bf16", "op": "mlp", "train": True, "rows": 8192, "width": 2048,
         "hidden": 5504, "act": "silu", "bias": False, "dtype": "bf16"},
        # The tokens of a time-frequency block in training: narrow, very many.
        {"name": "mlp training 129684x64 fp32", "op": "mlp", "train": True, "rows": 404 * 321, "width": 64,
         "hidden": 256, "act": "silu", "bias": True, "dtype": "fp32"},
    ]


def _between(rng, lo, hi):
    """A whole number of [lo, hi], its logarithm spread evenly."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """Mostly multiples of 32 (what models have), one in four any number."""
    c = _between(rng, lo, hi)
    return c if rng.random() < 0.25 else max(32, c // 32 * 32)


def draw(rng):
    op = rng.choice(["scan", "scan", "step", "mlp", "mlp"])
    dtype = rng.choice(["bf16", "fp32"])
    if op == "step":
        return {"op": op, "seqs": _between(rng, 1, 192), "width": _width(rng, 48, 4096), "dtype": dtype}
    train = rng.random() < 0.5
    if op == "mlp":
        width, hidden = _width(rng, 48, 4096), _width(rng, 64, 11008)
        # At most a third of the largest case's products.
        most = int(30e9 / (width * hidden) / (6 if dtype == "fp32" else 1))
        rows = _between(rng, 1, max(2, min(most, 131072, 60_000_000 // max(width, hidden))))
        return {"op": op, "train": train, "rows": rows, "width": width, "hidden": hidden,
                "act": rng.choice(["silu", "silu", "gelu"]), "bias": rng.random() < 0.5, "dtype": dtype}
    width = _width(rng, 48, 4096)
    rows = _between(rng, 64, min(max(65, 16_000_000 // width), 65536))
    seqs = min(_between(rng, 1, 400), max(1, rows // 2))
    ragged = rng.random() < 0.5
    if not ragged:
        rows = max(1, rows // seqs) * seqs
    return {"op": op, "train": train, "ragged": ragged, "rows": rows, "seqs": seqs, "width": width, "dtype": dtype}


_TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
_SCALE = 8.0  # of the recurrence's rate


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


def _pool(S, g):
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
    if op == "mlp":
        n, H = case["rows"], case["hidden"]
        st["x"] = rand(n, C)
        st["weight"] = rand(2 * H, C, scale=C ** -0.5)  # the value's rows, then the gate's
        st["bias"] = rand(2 * H, scale=0.1) if case["bias"] else None
        if case["train"]:
            st["dh"] = rand(n, H)
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
    st["x"] = rand(*lead, C)
    gates = rand(*lead, 2 * C)  # the rows of the gates' projection
    st["r"], st["i"] = gates[..., :C], gates[..., C:]
    st["z"] = rand(*lead, 2 * C)[..., C:]  # half of the in_proj output's rows
    # Decays of 0.9 to 0.999 where the gate is open.
    open_decay = torch.rand(C, generator=gpu, device="cuda") * 0.099 + 0.9
    st["rate"] = torch.log(torch.expm1(-torch.log(open_decay) / _SCALE))
    st["r_bias"], st["i_bias"] = rand(C, dtype=torch.float32, scale=0.3), rand(C, dtype=torch.float32, scale=0.3)
    if prompt:
        n_slots, st["slots"], st["fresh"] = _pool(S, host)
        st["state"] = rand(n_slots, C, dtype=torch.float32)
    else:
        st["dy"] = rand(*lead, C)
    return st


# -- the plain forms --------------------------------------------------------------------------


def _sigmoid(v):
    return 1 / (1 + torch.exp(-v))


def _softplus(v):
    return torch.where(v > 20, v, torch.log1p(torch.exp(torch.clamp(v, max=20))))


def _gates(st, shape):
    """Of each row: both gates, the decay, what 1 - a^2 is and the input's gain."""
    rho = _sigmoid(st["r"].reshape(shape).float() + st["r_bias"])
    iota = _sigmoid(st["i"].reshape(shape).float() + st["i_bias"])
    la = -_SCALE * _softplus(st["rate"]) * rho
    left = -torch.expm1(2 * la)
    return rho, iota, torch.exp(la), left, torch.sqrt(torch.clamp(left, min=1e-6))


def _running(a, b):
    """All h_t = a_t h_{t-1} + b_t along dim 0, from h = 0, by doubling: after the pass with distance d
    every row holds the sum over the 2 d rows up to it."""
    a, d = a.clone(), 1
    while d < a.shape[0]:
        b = torch.cat([b[:d], b[d:] + a[d:] * b[:-d]])
        a = torch.cat([a[:d], a[d:] * a[:-d]])
        d *= 2
    return b


def _scan(st):
    case = st["case"]
    C, rows, cu = case["width"], case["rows"], st["offsets"]
    t, shape = st["x"].dtype, st["x"].shape
    at = torch.arange(rows, device="cuda")
    seq = torch.searchsorted(cu[1:], at, right=True)
    on = (seq < cu.numel() - 1).float()[:, None]
    first = (at == cu[torch.clamp(seq, max=cu.numel() - 2)])[:, None]
    x, z = st["x"].reshape(-1, C).float(), st["z"].reshape(-1, C).float()
    rho, iota, a, left, gain = _gates(st, (-1, C))
    b = gain * iota * x
    if not case["train"]:
        slots = st["slots"].long()
        old = st["state"][slots]
        old[st["fresh"]] = 0
        b[cu[:-1]] += a[cu[:-1]] * old
    zero = torch.zeros((), device="cuda")
    linked = torch.where(first, zero, a)  # a sequence's first row sees nothing in front of it
    h = _running(linked, b)
    sig = _sigmoid(z)
    y = (h * z * sig * on).to(t).view(shape)
    if not case["train"]:
        st["state"][slots] = h[cu[1:] - 1]
        return {"y": y, "state": st["state"]}
    dy = st["dy"].reshape(-1, C).float() * on
    dz = dy * h * sig * (1 + z * (1 - sig))
    # g_t = dh_t + a_{t+1} g_{t+1}: the running sum of the rows turned round.
    nxt = torch.cat([linked[1:], torch.zeros_like(linked[:1])])
    g = torch.flip(_running(torch.flip(nxt, [0]), torch.flip(dy * z * sig, [0])), [0])
    before = torch.where(first, zero, torch.cat([torch.zeros_like(h[:1]), h[:-1]]))
    dla = g * a * before - torch.where(left > 1e-6, g * iota * x * a * a / gain, zero)
    dr = -_SCALE * _softplus(st["rate"]) * dla * rho * (1 - rho)
    di = g * gain * x * iota * (1 - iota)
    drate = -_SCALE * _sigmoid(st["rate"]).double() * (rho.double() * dla).sum(0)
    out = {"dx": g * gain * iota, "dr": dr, "di": di, "dz": dz}
    out = {k: (v * on).to(t).view(shape) for k, v in out.items()}
    return dict(out, y=y, drate=drate.float(), dr_bias=dr.double().sum(0).float(), di_bias=di.double().sum(0).float())


def _step(st):
    slots = st["slots"].long()
    rho, iota, a, left, gain = _gates(st, st["x"].shape)
    h = a * st["state"][slots] + gain * iota * st["x"].float()
    st["state"][slots] = h
    z = st["z"].float()
    return {"y": (h * z * _sigmoid(z)).to(st["x"].dtype), "state": st["state"]}


def _normal_cdf(v):
    return 0.5 * (1 + torch.erf(v * math.sqrt(0.5)))


def _mlp(st):
    case, t = st["case"], st["x"].dtype
    H, x, w = case["hidden"], st["x"].float(), st["weight"].float()
    both = x @ w.t()
    if case["bias"]:
        both = both + st["bias"].float()
    u, g = both[:, :H], both[:, H:]
    s = _sigmoid(g) if case["act"] == "silu" else _normal_cdf(g)
    h = (u * g * s).to(t)
    if not case["train"]:
        return {"h": h}
    dh = st["dh"].float()
    slope = s * (1 + g * (1 - s)) if case["act"] == "silu" else s + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    d = torch.cat([dh * g * s, dh * u * slope], 1)
    out = {"h": h, "dx": (d @ w).to(t), "dweight": (d.t() @ x).to(t)}
    if case["bias"]:
        out["dbias"] = d.double().sum(0).to(t)
    return out


# -- the package's calls ----------------------------------------------------------------------


def _leaf(v):
    return v.detach().requires_grad_()


def _own_scan(st):
    from semambaxlinoss_b200.gated_lru import gated_lru_scan

    if not st["case"]["train"]:
        y = gated_lru_scan(st["x"], st["r"], st["i"], st["rate"], z=st["z"], r_bias=st["r_bias"], i_bias=st["i_bias"],
                           rate_scale=_SCALE, cu_seqlens=st["cu"], state=st["state"], slots=st["slots"],
                           fresh=st["fresh"])
        return {"y": y, "state": st["state"]}
    names = ("x", "r", "i", "z", "rate", "r_bias", "i_bias")
    v = {k: _leaf(st[k]) for k in names}
    y = gated_lru_scan(v["x"], v["r"], v["i"], v["rate"], z=v["z"], r_bias=v["r_bias"], i_bias=v["i_bias"],
                       rate_scale=_SCALE, cu_seqlens=st["cu"])
    grads = torch.autograd.grad(y, [v[k] for k in names], st["dy"])
    return dict({"d" + k: g for k, g in zip(names, grads)}, y=y)


def _own_step(st):
    from semambaxlinoss_b200.gated_lru import gated_lru_step

    y = gated_lru_step(st["x"], st["r"], st["i"], st["rate"], st["state"], z=st["z"], r_bias=st["r_bias"],
                       i_bias=st["i_bias"], rate_scale=_SCALE, slots=st["slots"])
    return {"y": y, "state": st["state"]}


def _own_mlp(st):
    from semambaxlinoss_b200.gated_mlp import gated_linear

    case = st["case"]
    if not case["train"]:
        return {"h": gated_linear(st["x"], st["weight"], st["bias"], activation=case["act"])}
    names = ("x", "weight", "bias") if case["bias"] else ("x", "weight")
    v = {k: _leaf(st[k]) for k in names}
    h = gated_linear(v["x"], v["weight"], v.get("bias"), activation=case["act"])
    grads = torch.autograd.grad(h, [v[k] for k in names], st["dh"])
    return dict({"d" + k: g for k, g in zip(names, grads)}, h=h)


def run(state):
    op = state["case"]["op"]
    if own:
        return {"scan": _own_scan, "step": _own_step, "mlp": _own_mlp}[op](state)
    return {"scan": _scan, "step": _step, "mlp": _mlp}[op](state)


# -- what a pass cannot do without ------------------------------------------------------------


def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    C, op = case["width"], case["op"]
    if op == "mlp":
        n, H = case["rows"], case["hidden"]
        params = 2 * H * (C + (1 if case["bias"] else 0))
        if case["train"]:  # x, dh, the parameters; h, dx, the parameters' gradients
            return {"bytes": e * (2 * n * C + 2 * n * H + 2 * params), "flops": 12 * n * C * H + 30 * n * H}
        return {"bytes": e * (n * C + n * H + params), "flops": 4 * n * C * H + 10 * n * H}
    S = case["seqs"]
    if op == "step":  # x, r, i, z, y and the state, read and written
        return {"bytes": S * C * (5 * e + 8) + 12 * C, "flops": 35 * S * C}
    n = case["rows"] * C
    if case["train"]:  # x, r, i, z, dy; y, dx, dr, di, dz
        return {"bytes": 10 * n * e + 24 * C, "flops": 90 * n}
    return {"bytes": 5 * n * e + 8 * S * C + 12 * C, "flops": 35 * n}


# -- the definitions in 64 bits ---------------------------------------------------------------


def _exact_scan(case, st):
    """Step by step over sequences side by side, padded to the longest with rows that keep the state
    (decay one, no input) and take no gradient."""
    C, cu, train = case["width"], st["host_cu"], case["train"]
    length = [q - p for p, q in zip(cu[:-1], cu[1:])]
    S, L = len(length), max(max(length), 1)
    where = torch.full((L, S), case["rows"], dtype=torch.int64)
    for s in range(S):
        where[:length[s], s] = torch.arange(cu[s], cu[s + 1])
    where = where.cuda()
    live = (where < case["rows"])[..., None]

    def table(v):
        rows = v.double().reshape(-1, C)
        return torch.cat([rows, rows.new_zeros(1, C)])[where]

    def rows_of(v):
        out = v.new_zeros(case["rows"] + 1, C)
        out[where] = torch.where(live, v, torch.zeros_like(v[:1]))
        return out[:-1].view(st["x"].shape)

    x, z = table(st["x"]), table(st["z"])
    rho, iota = torch.sigmoid(table(st["r"]) + st["r_bias"].double()), torch.sigmoid(table(st["i"]) + st["i_bias"].double())
    rate = st["rate"].double()
    speed = _SCALE * torch.nn.functional.softplus(rate, threshold=40)
    a = torch.where(live, torch.exp(-speed * rho), torch.ones_like(x[:1]))
    left = torch.where(live, -torch.expm1(-2 * speed * rho), torch.ones_like(x[:1]))
    gain = torch.sqrt(torch.clamp(left, min=1e-6))
    h = x.new_zeros(S, C)
    if not train:
        h = torch.where(st["fresh"][:, None], h, st["state"].double()[st["slots"].long()])
    states = x.new_empty(L + 1, S, C)
    states[0] = h
    for t in range(L):
        h = a[t] * h + gain[t] * iota[t] * x[t]
        states[t + 1] = h
    silu = torch.nn.functional.silu(z)
    y = rows_of(states[1:] * silu)
    if not train:
        state = st["state"].double()
        state[st["slots"].long()] = h
        return {"y": y, "state": state}
    dy, sig = table(st["dy"]), torch.sigmoid(z)
    dz = dy * states[1:] * (sig + z * sig * (1 - sig))
    g, c = torch.empty_like(x), x.new_zeros(S, C)
    for t in range(L - 1, -1, -1):
        g[t] = dy[t] * silu[t] + c
        c = a[t] * g[t]
    da = g * states[:-1] - torch.where(left > 1e-6, a / gain, torch.zeros_like(a)) * g * iota * x
    drho = -speed * a * da
    dr, di = drho * rho * (1 - rho), g * gain * x * iota * (1 - iota)
    drate = (-_SCALE * a * da * rho).sum((0, 1)) * torch.sigmoid(rate)
    out = {"dx": g * gain * iota, "dr": dr, "di": di, "dz": dz}
    return dict({k: rows_of(v) for k, v in out.items()}, y=y, drate=drate, dr_bias=dr.sum((0, 1)),
                di_bias=di.sum((0, 1)))


def _exact_mlp(case, st):
    names = ("x", "weight", "bias") if case["bias"] else ("x", "weight")
    v = {k: st[k].double().requires_grad_(case["train"]) for k in names}
    both = torch.nn.functional.linear(v["x"], v["weight"], v.get("bias"))
    u, g = both.chunk(2, dim=-1)
    act = torch.nn.functional.silu if case["act"] == "silu" else torch.nn.functional.gelu
    h = u * act(g)
    if not case["train"]:
        return {"h": h}
    grads = torch.autograd.grad(h, [v[k] for k in names], st["dh"].double())
    return dict({"d" + k: d for k, d in zip(names, grads)}, h=h.detach())


def _exact_step(case, st):
    old = st["state"].double()
    slots = st["slots"].long()
    rho = torch.sigmoid(st["r"].double() + st["r_bias"].double())
    iota = torch.sigmoid(st["i"].double() + st["i_bias"].double())
    power = _SCALE * rho * torch.nn.functional.softplus(st["rate"].double(), threshold=40)
    gain = torch.sqrt(torch.clamp(-torch.expm1(-2 * power), min=1e-6))
    h = torch.exp(-power) * old[slots] + gain * iota * st["x"].double()
    old[slots] = h
    return {"y": h * torch.nn.functional.silu(st["z"].double()), "state": old}


def exact(case, seed):
    st = prepare(case, seed)
    return {"scan": _exact_scan, "step": _exact_step, "mlp": _exact_mlp}[case["op"]](case, st)
