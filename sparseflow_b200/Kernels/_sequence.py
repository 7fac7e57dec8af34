"""Argument checks shared by the sequence operators (causal_conv1d, selective_scan, block_norm).

A decoding step calls them for a few microseconds of GPU work, so they use what is cheapest to ask of a tensor.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd import forward_ad

from .. import _lib


def require_cuda(first: torch.Tensor, *others: Optional[torch.Tensor]) -> None:
    """All given tensors on one CUDA device, and none with a tangent: the kernels would drop it."""
    if forward_ad._current_level >= 0:
        _refuse_tangents(first, *others)
    if not first.is_cuda:
        raise RuntimeError("the sequence operators need CUDA tensors (there is no CPU path)")
    index = first.get_device()
    for t in others:
        if t is not None and t.get_device() != index:
            if not t.is_cuda:
                raise RuntimeError("the sequence operators need CUDA tensors (there is no CPU path)")
            raise ValueError(f"a tensor is on {t.device}, another on {first.device}")


def _refuse_tangents(*tensors: Optional[torch.Tensor]) -> None:
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError("the sequence operators have no forward-mode derivative")


def check_shape(name: str, t: torch.Tensor, shape) -> None:
    if t.shape != shape:
        raise ValueError(f"{name}: expected shape {list(shape)}, got {list(t.shape)}")


def check_dtype(name: str, t: torch.Tensor, dtype: torch.dtype) -> None:
    if t.dtype is not dtype:
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
    shape, stride = t.shape, t.stride()
    width = 1
    for k in range(1, inner + 1):
        if stride[-k] != width and shape[-k] != 1:
            if not t.numel():  # counts as contiguous whatever its strides are
                t = t.new_empty(shape)
                return t, t.stride(0), t.stride(-inner - 1)
            return rows_of(t.contiguous(), inner)
        width *= shape[-k]
    row = stride[-inner - 1] if shape[-inner - 1] > 1 else width
    if len(shape) == inner + 1:
        return t, 0, row
    return t, stride[0] if shape[0] > 1 else row * shape[1], row


def dense(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return t if t is None or t.is_contiguous() else t.contiguous()


def needs_grad(*tensors: Optional[torch.Tensor]) -> bool:
    if not torch.is_grad_enabled():
        return False
    for t in tensors:
        if t is not None and t.requires_grad:
            return True
    return False


class _NoGradient(torch.autograd.Function):
    """The result of a function without a gradient as a part of the graph, so that a backward pass that comes to it
    raises instead of passing over it."""

    @staticmethod
    def forward(ctx, fn, *args):
        ctx.name = fn.__name__
        return fn(*args)

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError(f"{ctx.name} has no gradient: run sequences through the prompt's function to train")


without_gradient = _NoGradient.apply


# Tensors that a kernel has written in place count as changed, so that a backward pass that had saved one raises.
written = torch._C._increment_version


def layout(t: Optional[torch.Tensor]):
    """What the checks of a call depend on, as a key of calls that have passed them."""
    return None if t is None else (t.shape, t.stride(), t.dtype)


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
