"""Argument checks and batch description shared by the selective state operators."""
from __future__ import annotations

import torch

TYPES = (torch.float32, torch.bfloat16)
_ROW_MAX = 2 ** 31


def rows_of(t: torch.Tensor, width: int, inner: int = 1) -> tuple[torch.Tensor, int]:
    """``t`` (rows, ...) or (S, L, ...) with ``inner`` dimensions of ``width`` elements in all as
    (tensor, row stride): read in place where its rows lie at one stride with contiguous
    elements, else a contiguous copy."""
    if t.is_contiguous():
        return t, width
    shape, stride = t.shape, t.stride()
    if (stride[-1] == 1 or shape[-1] == 1) and (inner == 1 or stride[-2] == shape[-1] or shape[-2] == 1):
        if len(shape) == 1 + inner:
            ld = stride[0] if shape[0] > 1 else width
        elif shape[1] == 1:
            ld = stride[0] if shape[0] > 1 else width
        elif shape[0] == 1 or stride[0] == shape[1] * stride[1]:
            ld = stride[1]
        else:
            ld = 0
        if width <= ld < _ROW_MAX:
            return t, ld
    return t.contiguous(), width


def check_same(op: str, name: str, t: torch.Tensor, shape, dtypes, dev: int) -> None:
    """``dev``: the GPU's number (``Tensor.get_device``)."""
    if t.shape != shape or t.dtype not in dtypes or t.get_device() != dev:
        want = " or ".join(str(d).replace("torch.", "") for d in dtypes)
        raise ValueError(f"{op}: {name} must be {want} {tuple(shape)} on cuda:{dev}, got {t.dtype} {tuple(t.shape)} "
                         f"on {t.device}")


def batch(op: str, x: torch.Tensor, cu_seqlens) -> tuple[int, int, int]:
    """(S, rows, L) of x (S, L, C), or of packed x (rows, C) with cu_seqlens (S + 1)."""
    if not x.is_cuda:
        raise RuntimeError(f"{op} requires CUDA tensors.")
    if x.dtype not in TYPES:
        raise ValueError(f"{op}: unsupported dtype {x.dtype}")
    if cu_seqlens is None:
        if x.dim() != 3:
            raise ValueError(f"{op}: x must be (batch, length, channels), or (rows, channels) with cu_seqlens, got "
                             f"{tuple(x.shape)}")
        return x.shape[0], x.shape[0] * x.shape[1], x.shape[1]
    if x.dim() != 2:
        raise ValueError(f"{op}: packed x must be (rows, channels), got {tuple(x.shape)}")
    if (cu_seqlens.dtype != torch.int32 or cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 1
            or cu_seqlens.device != x.device or not cu_seqlens.is_contiguous()):
        raise ValueError(f"{op}: cu_seqlens must be contiguous int32 (sequences + 1,) on {x.device}, got "
                         f"{cu_seqlens.dtype} {tuple(cu_seqlens.shape)} on {cu_seqlens.device}")
    return cu_seqlens.shape[0] - 1, x.shape[0], 0


def set_pool(op: str, a, S: int, dev: int, state, shape, dtype, slots, fresh) -> None:
    """Checks the state pool (entries of ``shape``) and its index and fills the argument struct."""
    if state is None:
        if slots is not None or fresh is not None:
            raise ValueError(f"{op}: slots / fresh without a state")
        return
    if (state.shape[1:] != shape or state.dtype != dtype or state.get_device() != dev or not state.is_contiguous()):
        raise ValueError(f"{op}: the state must be contiguous {str(dtype)[6:]} (entries, "
                         f"{', '.join(map(str, shape))}) on cuda:{dev}, got {state.dtype} {tuple(state.shape)} on "
                         f"{state.device}")
    if state.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{op}: the state is updated in place and cannot require a gradient")
    n = state.shape[0]
    if n == 0:
        # Every slot is behind an empty pool; the library takes a pool of none as "no state".
        raise ValueError(f"{op}: the state has no entries")
    if slots is None:
        if n < S:
            raise ValueError(f"{op}: {n} state entries for {S} sequences")
    else:
        if slots.shape != (S,) or slots.dtype != torch.int32 or slots.get_device() != dev or not slots.is_contiguous():
            raise ValueError(f"{op}: slots must be contiguous int32 ({S},) on cuda:{dev}, got {slots.dtype} "
                             f"{tuple(slots.shape)} on {slots.device}")
        a.slots = slots.data_ptr()
    if fresh is not None:
        if fresh.shape != (S,) or fresh.dtype != torch.bool or fresh.get_device() != dev or not fresh.is_contiguous():
            raise ValueError(f"{op}: fresh must be contiguous bool ({S},) on cuda:{dev}, got {fresh.dtype} "
                             f"{tuple(fresh.shape)} on {fresh.device}")
        a.fresh = fresh.data_ptr()
    a.n_slots, a.state = n, state.data_ptr()
