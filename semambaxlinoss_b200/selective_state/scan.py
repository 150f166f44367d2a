"""Selective state scan (``semx_state_scan_fwd/bwd``, ``semx_state_step``).

Per channel c with N modes, channels in G groups that share B and C::

    d    = softplus(dt + dt_bias)          (dt + dt_bias without dt_softplus)
    h[n] = exp(d A[c, n]) h[n] + d x B[n]
    y    = (sum_n C[n] h[n] + D x) silu(z) (no gate without z)

Next to :func:`~semambaxlinoss_b200.selective_lru.fused_selective_lru_real` (gain "mamba"),
whose operands are fp32 with the step already evaluated, the operands here are the
projections' own outputs (bf16 or fp32, at their row strides), sequences may be packed and
may keep their state in a pool between calls, and there is a form for single tokens. The
state is fp32 throughout.
"""
from __future__ import annotations

import torch

from .. import _lib
from ._batch import TYPES, batch, check_same, rows_of, set_pool

MAX_MODES = 128
_F32 = (torch.float32,)


def _check(op, x, dt, A, B, C, D, z, dt_bias):
    """Shapes and types; returns (channels, modes, groups)."""
    shape, dtype, dev = x.shape, x.dtype, x.get_device()
    ch, Ashape = shape[-1], A.shape
    if len(Ashape) != 2 or Ashape[0] != ch or not 1 <= Ashape[1] <= MAX_MODES:
        raise ValueError(f"{op}: A must be ({ch}, modes) with 1 to {MAX_MODES} modes, got {tuple(Ashape)}")
    N, Bshape = Ashape[1], B.shape
    grouped = len(Bshape) == len(shape) + 1
    G = Bshape[-2] if grouped else 1
    if G < 1 or ch % G:
        raise ValueError(f"{op}: {ch} channels do not fall into {G} groups")
    want = shape[:-1] + ((G, N) if grouped else (N,))
    types = _F32 if dtype == torch.float32 else TYPES
    # One expression for the calls that are right, which a decoding loop makes thousands of.
    if not (dt.shape == shape and Bshape == want and C.shape == want and dt.dtype in types and A.dtype in TYPES
            and B.dtype == dtype and C.dtype == dtype and dt.get_device() == dev and A.get_device() == dev
            and B.get_device() == dev and C.get_device() == dev
            and (z is None or (z.shape == shape and z.dtype == dtype and z.get_device() == dev))
            and (D is None or (D.shape == (ch,) and D.dtype in TYPES and D.get_device() == dev))
            and (dt_bias is None or (dt_bias.shape == (ch,) and dt_bias.dtype in TYPES and dt_bias.get_device() == dev))):
        check_same(op, "A", A, Ashape, TYPES, dev)
        check_same(op, "dt", dt, shape, types, dev)
        for name, t, s in (("B", B, want), ("C", C, want), ("z", z, shape)):
            if t is not None:
                check_same(op, name, t, s, (dtype,), dev)
        for name, t in (("D", D), ("dt_bias", dt_bias)):
            if t is not None:
                check_same(op, name, t, (ch,), TYPES, dev)
    return ch, N, G


def _grads_wanted(x, dt, A, B, C, D, z, dt_bias):
    return torch.is_grad_enabled() and (
        x.requires_grad or dt.requires_grad or A.requires_grad or B.requires_grad or C.requires_grad
        or (D is not None and D.requires_grad) or (z is not None and z.requires_grad)
        or (dt_bias is not None and dt_bias.requires_grad))


def _args(x, dt, A, B, C, D, z, dt_bias, softplus, S, rows, L, cu, N, G):
    """The argument struct, and what has to outlive the call."""
    ch = A.shape[0]
    inner = B.dim() - x.dim() + 1  # (groups, modes) or (modes,)
    x, ldx = rows_of(x, ch)
    dt, ldd = rows_of(dt, ch)
    B, ldb = rows_of(B, G * N, inner)
    C, ldc = rows_of(C, G * N, inner)
    a = _lib.new_args(_lib.SemxStateScanArgs)
    a.softplus, a.bf16, a.dt_bf16 = softplus, x.dtype == torch.bfloat16, dt.dtype == torch.bfloat16
    a.S, a.rows, a.L, a.C, a.N, a.G = S, rows, L, ch, N, G
    a.ldx, a.lddt, a.ldb, a.ldc = ldx, ldd, ldb, ldc
    a.x, a.dt, a.A, a.B, a.Cm = x.data_ptr(), dt.data_ptr(), A.data_ptr(), B.data_ptr(), C.data_ptr()
    if z is not None:
        z, a.ldz = rows_of(z, ch)
        a.z = z.data_ptr()
    if D is not None:
        a.D = D.data_ptr()
    if dt_bias is not None:
        a.dt_bias = dt_bias.data_ptr()
    if cu is not None:
        a.cu_seqlens = cu.data_ptr()
    return a, (x, dt, B, C, z)


class _StateScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, dt, A, B, C, D, z, dt_bias, softplus, S, rows, L, cu, N, G):
        A32, D32, b32 = _lib.param32(A), _lib.param32(D), _lib.param32(dt_bias)
        a, kept = _args(x, dt, A32, B, C, D32, z, b32, softplus, S, rows, L, cu, N, G)
        dev = x.device
        y = x.new_empty(x.shape)
        v = None if z is None else x.new_empty(x.shape, dtype=torch.float32)
        ckpt = _lib.scratch(_lib.load().semx_state_scan_ckpt_bytes(a), x)
        a.y, a.v, a.ckpt = y.data_ptr(), _lib.ptr(v), ckpt.data_ptr()
        nbytes = _lib.load().semx_state_scan_workspace_bytes(a, 0)
        ws = _lib.scratch(nbytes, x) if nbytes else None
        a.workspace = _lib.ptr(ws)
        _lib.call("semx_state_scan_fwd", a, dev)
        xr, dr, Br, Cr, zr = kept
        ctx.save_for_backward(xr, dr, A32, Br, Cr, D32, zr, b32, v, ckpt, cu)
        ctx.cfg = (softplus, S, rows, L, N, G, B.shape, [None if t is None else t.dtype for t in (A, D, dt_bias)])
        return y

    @staticmethod
    @_lib.once_differentiable
    def backward(ctx, dy):
        x, dt, A, B, C, D, z, bias, v, ckpt, cu = ctx.saved_tensors
        softplus, S, rows, L, N, G, Bshape, (Adt, Ddt, bdt) = ctx.cfg
        a, kept = _args(x, dt, A, B, C, D, z, bias, softplus, S, rows, L, cu, N, G)
        dev = x.device
        dy = _lib.as_rows(dy, x.dtype)
        dx, ddt = x.new_empty(x.shape), dt.new_empty(x.shape)
        dz = None if z is None else x.new_empty(x.shape)
        dB, dC = x.new_empty(Bshape), x.new_empty(Bshape)
        need = ctx.needs_input_grad
        dA = torch.empty_like(A) if need[2] else None
        dD = torch.empty_like(D) if D is not None and need[5] else None
        db = torch.empty_like(bias) if bias is not None and need[7] else None
        a.v, a.ckpt, a.dy, a.dx, a.ddt, a.dz = (_lib.ptr(v), ckpt.data_ptr(), dy.data_ptr(), dx.data_ptr(),
                                                ddt.data_ptr(), _lib.ptr(dz))
        a.dB, a.dC, a.dA, a.dD, a.ddt_bias = dB.data_ptr(), dC.data_ptr(), _lib.ptr(dA), _lib.ptr(dD), _lib.ptr(db)
        ws = _lib.scratch(_lib.load().semx_state_scan_workspace_bytes(a, 1), x)
        a.workspace = ws.data_ptr()
        _lib.call("semx_state_scan_bwd", a, dev)

        return (dx, ddt, _lib.cast(dA, Adt), dB, dC, _lib.cast(dD, Ddt), dz, _lib.cast(db, bdt), None, None, None, None,
                None, None, None)


def selective_state_scan(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                         D: torch.Tensor | None = None, z: torch.Tensor | None = None,
                         dt_bias: torch.Tensor | None = None, dt_softplus: bool = True,
                         cu_seqlens: torch.Tensor | None = None, state: torch.Tensor | None = None,
                         slots: torch.Tensor | None = None, fresh: torch.Tensor | None = None) -> torch.Tensor:
    """Selective scan of the sequences in ``x``; y has x's shape and type.

    x, dt, z: (S, L, C), or packed (rows, C) with ``cu_seqlens`` (see
    :func:`~semambaxlinoss_b200.selective_state.short_conv` for the batch, and for state, slots
    and fresh). B, C: (S, L, N) or (S, L, G, N) (packed: (rows, N) or (rows, G, N)); A (C, N),
    N up to 128; D, dt_bias (C,). x, z, B and C are of one type, bf16 or fp32; dt may be fp32
    beside bf16. Rows may lie at any stride.

    Training: gradients flow to every operand, every sequence starts from zeros; the forward
    keeps the state of every 8th step and, with z, the value in front of the gate, both in
    fp32. Prompts: ``state`` (entries, C, N) fp32 is read and updated in place; refused
    while a gradient is wanted."""
    op = "selective_state_scan"
    S, rows, L = batch(op, x, cu_seqlens)
    if _lib.in_dual_level():
        _lib.refuse_tangents(op, x, dt, A, B, C, D, z, dt_bias, state)
    ch, N, G = _check(op, x, dt, A, B, C, D, z, dt_bias)
    softplus = int(bool(dt_softplus))
    if _grads_wanted(x, dt, A, B, C, D, z, dt_bias):
        if state is not None:
            raise ValueError(f"{op}: a state is for inference; the call wants gradients")
        if slots is not None or fresh is not None:
            raise ValueError(f"{op}: slots / fresh without a state")
        return _StateScan.apply(x, dt, A, B, C, D, z, dt_bias, softplus, S, rows, L, cu_seqlens, N, G)
    A, D, dt_bias = _lib.param32(A), _lib.param32(D), _lib.param32(dt_bias)
    a, kept = _args(x, dt, A, B, C, D, z, dt_bias, softplus, S, rows, L, cu_seqlens, N, G)
    dev = x.device
    set_pool(op, a, S, x.get_device(), state, (ch, N), torch.float32, slots, fresh)
    y = x.new_empty(x.shape)
    a.y = y.data_ptr()
    nbytes = _lib.load().semx_state_scan_workspace_bytes(a, 0)
    ws = _lib.scratch(nbytes, x) if nbytes else None
    a.workspace = _lib.ptr(ws)
    _lib.call("semx_state_scan_fwd", a, dev)
    return y


def selective_state_step(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                         state: torch.Tensor, D: torch.Tensor | None = None, z: torch.Tensor | None = None,
                         dt_bias: torch.Tensor | None = None, dt_softplus: bool = True,
                         slots: torch.Tensor | None = None) -> torch.Tensor:
    """One token of every sequence: x, dt, z (S, C), B, C (S, N) or (S, G, N) -> y (S, C);
    ``state`` (entries, C, N) fp32 is updated in place. Slots as in
    :func:`~semambaxlinoss_b200.selective_state.short_conv`. Not differentiable."""
    op = "selective_state_step"
    if not x.is_cuda:
        raise RuntimeError(f"{op} requires CUDA tensors.")
    if x.dim() != 2 or x.dtype not in TYPES:
        raise ValueError(f"{op}: x must be fp32 or bf16 (sequences, channels), got {x.dtype} {tuple(x.shape)}")
    if state is None:
        raise ValueError(f"{op}: a state is needed")
    if _lib.in_dual_level():
        _lib.refuse_tangents(op, x, dt, A, B, C, state, D, z, dt_bias)
    ch, N, G = _check(op, x, dt, A, B, C, D, z, dt_bias)
    if _grads_wanted(x, dt, A, B, C, D, z, dt_bias):
        raise ValueError(f"{op}: a state is for inference; the call wants gradients")
    S = x.shape[0]
    A, D, dt_bias = _lib.param32(A), _lib.param32(D), _lib.param32(dt_bias)
    a, kept = _args(x, dt, A, B, C, D, z, dt_bias, int(bool(dt_softplus)), S, S, 1, None, N, G)
    set_pool(op, a, S, x.get_device(), state, (ch, N), torch.float32, slots, None)
    y = x.new_empty(x.shape)
    a.y = y.data_ptr()
    _lib.call("semx_state_step", a, x.device)
    return y
