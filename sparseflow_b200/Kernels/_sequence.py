"""Argument checks shared by the sequence operators (causal_conv1d, selective_scan, block_norm)."""
from __future__ import annotations

from typing import Optional

import torch

from .. import _lib


def require_cuda(**tensors: Optional[torch.Tensor]) -> torch.device:
    """All given tensors on one CUDA device; returns it."""
    device = None
    for name, t in tensors.items():
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError(f"{name}: the sequence operators need CUDA tensors (there is no CPU path)")
        if device is None:
            device = t.device
        elif t.device != device:
            raise ValueError(f"{name} is on {t.device}, the others on {device}")
    return device


def check_shape(name: str, t: torch.Tensor, shape) -> None:
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name}: expected shape {list(shape)}, got {list(t.shape)}")


def check_dtype(name: str, t: torch.Tensor, dtype: torch.dtype) -> None:
    if t.dtype != dtype:
        raise TypeError(f"{name}: expected {dtype}, got {t.dtype}")


def check_offsets(seq_offsets: Optional[torch.Tensor], x: torch.Tensor):
    """(number of sequences, rows: of each or in all, packed) of x [B, L, dim], or [total, dim] with offsets."""
    if seq_offsets is None:
        if x.dim() != 3:
            raise ValueError(f"x: expected [batch, length, dim], or [total, dim] with seq_offsets; got {list(x.shape)}")
        return x.shape[0], x.shape[1], False
    if x.dim() != 2:
        raise ValueError(f"x: expected [total, dim] with seq_offsets, got {list(x.shape)}")
    check_dtype("seq_offsets", seq_offsets, torch.int32)
    if seq_offsets.dim() != 1 or seq_offsets.numel() < 1 or not seq_offsets.is_contiguous():
        raise ValueError("seq_offsets: expected n_seq + 1 contiguous offsets")
    return seq_offsets.numel() - 1, x.shape[0], True


def rows_of(t: torch.Tensor, inner: int = 1):
    """The tensor with its last `inner` dimensions contiguous (copied only where they are not) and its batch and
    row strides; the strides of dimensions of one entry, which may be anything, are those of a contiguous tensor."""
    width = 1
    for k in range(1, inner + 1):
        if t.shape[-k] != 1 and t.stride(-k) != width:
            t = t.contiguous()
            break
        width *= t.shape[-k]
    width = 1
    for k in range(1, inner + 1):
        width *= t.shape[-k]
    row = t.stride(-inner - 1) if t.shape[-inner - 1] > 1 else width
    if t.dim() == inner + 1:
        return t, 0, row
    return t, t.stride(0) if t.shape[0] > 1 else row * t.shape[1], row


def needs_grad(*tensors: Optional[torch.Tensor]) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def check_state_indices(state_indices: Optional[torch.Tensor], rows: int, slots: int) -> None:
    if state_indices is None:
        if slots < rows:
            raise ValueError(f"state: {slots} slots for {rows} rows and no state_indices")
        return
    check_dtype("state_indices", state_indices, torch.int32)
    check_shape("state_indices", state_indices, (rows,))
    if not state_indices.is_contiguous():
        raise ValueError("state_indices: expected a contiguous tensor")


call_on = _lib.call_on
