"""Short causal convolution along a sequence, one filter per channel (csrc/causal_conv1d.cu).

The mixer of neighbouring tokens that comes before the selective state space scan. No counterpart in the
reference: it extends the framework's temporal operators (the multi-step LIF) by a learned one.
"""
from __future__ import annotations

from typing import Optional

import torch

from .. import _lib
from ._sequence import (call_on, check_dtype, check_offsets, check_shape, check_state_indices, dense, layout, needs_grad, ptr,
                        require_cuda, rows_of, without_gradient, written)

_ACTIVATIONS = {None: False, "silu": True}


def _check(x, weight, bias, activation):
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation: expected None or 'silu', got {activation!r}")
    dim = x.shape[-1]
    if weight.dim() != 2 or weight.shape[0] != dim or not 2 <= weight.shape[1] <= 8:
        raise ValueError(f"weight: expected [{dim}, width] with 2 to 8 taps, got {list(weight.shape)}")
    if bias is not None:
        check_shape("bias", bias, (dim,))
        check_dtype("bias", bias, weight.dtype)
    return dim, weight.shape[1]


def _forward(x, weight, bias, initial_state, seq_offsets, silu, want_final):
    n_seq, length, packed = check_offsets(seq_offsets, x)
    dim, width = weight.shape
    x, batch, row = rows_of(x)
    y = x.new_empty(x.shape)
    final = torch.empty(n_seq, width - 1, dim, dtype=x.dtype, device=x.device) if want_final else None
    desc = _lib.causal_conv1d_desc(length, batch, row, n_seq, dim, width, silu, x.dtype, weight.dtype, packed)
    call_on(x.get_device(), "sf_causal_conv1d", ptr(x), ptr(weight), ptr(bias), ptr(initial_state), ptr(seq_offsets), ptr(y),
            ptr(final), desc)
    return y, final, desc, x


class _CausalConv1d(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, initial_state, seq_offsets, silu, want_final):
        y, final, ctx.desc, x = _forward(x, weight, bias, initial_state, seq_offsets, silu, want_final)
        ctx.save_for_backward(x, weight, bias, initial_state, seq_offsets)
        ctx.set_materialize_grads(False)
        return y, final

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dfinal):
        x, weight, bias, initial_state, seq_offsets = ctx.saved_tensors
        dy = torch.zeros(x.shape, dtype=x.dtype, device=x.device) if dy is None else dense(dy)
        dfinal = dense(dfinal)
        dx = x.new_empty(x.shape)
        dweight = torch.empty_like(weight)
        dbias = None if bias is None else torch.empty_like(bias)
        dinit = torch.empty_like(initial_state) if initial_state is not None and ctx.needs_input_grad[3] else None
        nbytes = _lib.load().sf_causal_conv1d_backward_workspace_size(ctx.desc)
        ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=x.device)
        call_on(x.get_device(), "sf_causal_conv1d_backward", ptr(x), ptr(weight), ptr(bias), ptr(initial_state),
                ptr(seq_offsets), ptr(dy), ptr(dfinal), ptr(dx), ptr(dweight), ptr(dbias), ptr(dinit), ctx.desc,
                ptr(ws), nbytes)
        return dx, dweight, dbias, dinit, None, None, None


def causal_conv1d(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                  activation: Optional[str] = None, initial_state: Optional[torch.Tensor] = None,
                  seq_offsets: Optional[torch.Tensor] = None, return_final_state: bool = False):
    """y[t] = act(bias + sum_k weight[:, k] x[t - (width - 1) + k]) for every channel.

    x: [batch, length, dim], or [total, dim] of packed sequences with ``seq_offsets`` (int32 [n_seq + 1] on the
    device, from 0 to total; sequences may be empty). Rows may be slices of wider rows. weight [dim, width], 2 to 8
    taps; bias [dim] in the weight's type. ``initial_state`` [n_seq, width - 1, dim] in x's type holds the rows
    before each sequence, oldest first (zeros if None). Returns y, or (y, final_state) where the final state is the
    next call's initial one. Differentiable once, in x, weight, bias and the initial state.
    """
    require_cuda(x, weight, bias, initial_state, seq_offsets)
    dim, width = _check(x, weight, bias, activation)
    n_seq, _, _ = check_offsets(seq_offsets, x)
    if initial_state is not None:
        check_shape("initial_state", initial_state, (n_seq, width - 1, dim))
        check_dtype("initial_state", initial_state, x.dtype)
        initial_state = dense(initial_state)
    weight, bias = dense(weight), dense(bias)
    silu = _ACTIVATIONS[activation]
    if needs_grad(x, weight, bias, initial_state):
        y, final = _CausalConv1d.apply(x, weight, bias, initial_state, seq_offsets, silu, return_final_state)
    else:
        y, final, _, _ = _forward(x, weight, bias, initial_state, seq_offsets, silu, return_final_state)
    return (y, final) if return_final_state else y


def causal_conv1d_update(x: torch.Tensor, state: torch.Tensor, weight: torch.Tensor,
                         bias: Optional[torch.Tensor] = None, activation: Optional[str] = None,
                         state_indices: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One more token: x [rows, dim] -> y [rows, dim]; ``state`` [slots, width - 1, dim] is shifted in place.

    Row i uses slot ``state_indices[i]`` (int32 on the device, distinct), or slot i without indices. A row whose
    index is no slot (-1, say) is padding: its y is 0 and no state changes. Not differentiable: where an input asks
    for a gradient, a backward pass through y raises.
    """
    require_cuda(x, state, weight, bias, state_indices)
    if torch.is_grad_enabled() and (x.requires_grad or state.requires_grad or weight.requires_grad
                                    or (bias is not None and bias.requires_grad)):
        return without_gradient(causal_conv1d_update, x, state, weight, bias, activation, state_indices)
    key = (x.shape, x.stride(), x.dtype, state.shape, state.stride(), state.dtype, weight.shape, weight.stride(),
           weight.dtype, layout(bias), layout(state_indices), activation)
    desc = _update_plans.get(key)
    if desc is None:
        x, weight, bias, desc = _update_plan(x, state, weight, bias, activation, state_indices, key)
    y = x.new_empty(x.shape)
    call_on(x.get_device(), "sf_causal_conv1d_update", x.data_ptr(), state.data_ptr(), weight.data_ptr(), ptr(bias),
            ptr(state_indices), y.data_ptr(), state.shape[0], desc)
    written((state,))
    return y


# Descriptors of the layouts that single-token calls have come with, where nothing had to be copied: a decoding loop's
# next call with the same layouts has passed its checks.
_update_plans: dict = {}


def _update_plan(x, state, weight, bias, activation, state_indices, key):
    """Checks a call and returns its operands as the kernel reads them and its descriptor."""
    if x.dim() != 2:
        raise ValueError(f"x: expected [rows, dim], got {list(x.shape)}")
    dim, width = _check(x, weight, bias, activation)
    if state.dim() != 3 or not state.is_contiguous():
        raise ValueError("state: expected a contiguous [slots, width - 1, dim] tensor")
    check_shape("state", state, (state.shape[0], width - 1, dim))
    check_dtype("state", state, x.dtype)
    check_state_indices(state_indices, x.shape[0], state.shape[0])
    given = (x, weight, bias)
    weight, bias = dense(weight), dense(bias)
    x, _, row = rows_of(x)
    desc = _lib.causal_conv1d_desc(1, 0, row, x.shape[0], dim, width, _ACTIVATIONS[activation], x.dtype, weight.dtype,
                                   False)
    if all(a is b for a, b in zip((x, weight, bias), given)):
        if len(_update_plans) >= 512:
            _update_plans.clear()
        _update_plans[key] = desc
    return x, weight, bias, desc
