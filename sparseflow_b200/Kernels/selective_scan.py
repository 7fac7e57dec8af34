"""Selective state space scan (csrc/selective_scan.cu): the learned, linear counterpart of the LIF recurrence.

Where a LIF neuron leaks its membrane by a fixed factor and fires, a state space channel keeps several states that
decay by factors chosen by the input (through dt) and reads them out by inner products. No counterpart in the
reference.
"""
from __future__ import annotations

from typing import Optional

import torch

from .. import _lib
from ._sequence import (call_on, check_dtype, check_offsets, check_shape, check_state_indices, dense, layout, needs_grad, ptr,
                        require_cuda, rows_of, without_gradient, written)

_MAX_STATE = 128


def _check(x, dt, A, B, C, D, z, dt_bias):
    """Checks the operands against x's leading dimensions; B and C get their group dimension. Returns
    (B, C, dim, state, groups)."""
    shape, kind = x.shape, x.dtype
    dim = shape[-1]
    if A.dim() != 2 or A.shape[0] != dim or not 1 <= A.shape[1] <= _MAX_STATE:
        raise ValueError(f"A: expected [{dim}, state] with 1 to {_MAX_STATE} states, got {list(A.shape)}")
    state = A.shape[1]
    if B.dim() == len(shape):
        B = B.unsqueeze(-2)
    if C.dim() == len(shape):
        C = C.unsqueeze(-2)
    groups = B.shape[-2] if B.dim() >= 2 else 0
    if groups < 1 or dim % groups:
        raise ValueError(f"B: {groups} groups do not divide {dim} channels")
    inner = (*shape[:-1], groups, state)
    check_shape("B", B, inner)
    check_shape("C", C, inner)
    check_shape("dt", dt, shape)
    check_dtype("dt", dt, kind)
    check_dtype("B", B, kind)
    check_dtype("C", C, kind)
    if z is not None:
        check_dtype("z", z, kind)
        check_shape("z", z, shape)
    if D is not None:
        check_shape("D", D, (dim,))
    if dt_bias is not None:
        check_shape("dt_bias", dt_bias, (dim,))
    return B, C, dim, state, groups


def _float(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """Parameters are read in 32 bits; autograd sees the cast."""
    return t if t is None or (t.dtype is torch.float32 and t.is_contiguous()) else t.float().contiguous()


def _strided(x, dt, z, B, C):
    """The operands as the kernels read them, and their (batch, row) strides one after another."""
    x, x0, x1 = rows_of(x)
    dt, t0, t1 = rows_of(dt)
    z0 = z1 = 0
    if z is not None:
        z, z0, z1 = rows_of(z)
    B, b0, b1 = rows_of(B, 2)
    C, c0, c1 = rows_of(C, 2)
    return x, dt, z, B, C, (x0, x1, t0, t1, z0, z1, b0, b1, c0, c1)


def _forward(x, dt, A, B, C, D, z, dt_bias, initial_state, seq_offsets, softplus, want_final, want_checkpoints):
    n_seq, length, packed = check_offsets(seq_offsets, x)
    dim, state = A.shape
    groups = B.shape[-2]
    x, dt, z, B, C, strides = _strided(x, dt, z, B, C)
    desc = _lib.selective_scan_desc(length, strides, n_seq, dim, state, groups, softplus, x.dtype, packed)
    lib = _lib.load()
    y = x.new_empty(x.shape)
    final = A.new_empty((n_seq, dim, state)) if want_final else None
    ck = None
    if want_checkpoints:
        ck = A.new_empty(lib.sf_selective_scan_checkpoint_bytes(desc) // 4)
    nbytes = lib.sf_selective_scan_workspace_size(desc)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device) if nbytes else None
    call_on(x.get_device(), "sf_selective_scan", ptr(x), ptr(dt), ptr(A), ptr(B), ptr(C), ptr(D), ptr(z), ptr(dt_bias),
            ptr(initial_state), ptr(seq_offsets), ptr(y), ptr(final), ptr(ck), desc, ptr(ws), nbytes)
    return y, final, ck, desc, (x, dt, z, B, C)


class _SelectiveScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, dt, A, B, C, D, z, dt_bias, initial_state, seq_offsets, softplus, want_final):
        y, final, ck, ctx.desc, (x, dt, z, B, C) = _forward(x, dt, A, B, C, D, z, dt_bias, initial_state, seq_offsets,
                                                            softplus, want_final, True)
        ctx.save_for_backward(x, dt, A, B, C, D, z, dt_bias, seq_offsets, ck)
        ctx.state_shape = None if initial_state is None else initial_state.shape
        ctx.set_materialize_grads(False)
        return y, final

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dfinal):
        x, dt, A, B, C, D, z, dt_bias, seq_offsets, ck = ctx.saved_tensors

        def like(t):
            return None if t is None else t.new_empty(t.shape)

        dy = torch.zeros(x.shape, dtype=x.dtype, device=x.device) if dy is None else dense(dy)
        dfinal = dense(dfinal)
        dx, ddt, dA, dB, dC, dD, dz, dbias = (like(t) for t in (x, dt, A, B, C, D, z, dt_bias))
        dinit = None
        if ctx.state_shape is not None and ctx.needs_input_grad[8]:
            dinit = A.new_empty(ctx.state_shape)
        nbytes = _lib.load().sf_selective_scan_backward_workspace_size(ctx.desc)
        ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=x.device)
        call_on(x.get_device(), "sf_selective_scan_backward", ptr(x), ptr(dt), ptr(A), ptr(B), ptr(C), ptr(D), ptr(z),
                ptr(dt_bias), ptr(seq_offsets), ptr(ck), ptr(dy), ptr(dfinal), ptr(dx), ptr(ddt), ptr(dA), ptr(dB),
                ptr(dC), ptr(dD), ptr(dz), ptr(dbias), ptr(dinit), ctx.desc, ptr(ws), nbytes)
        return dx, ddt, dA, dB, dC, dD, dz, dbias, dinit, None, None, None


def selective_scan(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                   D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None,
                   dt_bias: Optional[torch.Tensor] = None, dt_softplus: bool = True,
                   initial_state: Optional[torch.Tensor] = None, seq_offsets: Optional[torch.Tensor] = None,
                   return_final_state: bool = False):
    """h_t = exp(dt_t A) h_(t-1) + dt_t x_t B_t, y_t = (C_t . h_t + D x_t) silu(z_t), channel by channel.

    x, dt, z: [batch, length, dim], or [total, dim] of packed sequences with ``seq_offsets`` (int32 [n_seq + 1] on
    the device, from 0 to total; sequences may be empty; up to 65535 of them either way); B, C: the same leading dimensions and [state] or
    [groups, state] (channel d reads group d // (dim / groups)), all of x's type. Rows may be slices of wider rows.
    A [dim, state], D, dt_bias [dim] are read in 32 bits. dt is softplus(dt + dt_bias), or dt + dt_bias without
    ``dt_softplus``. States are fp32 [n_seq, dim, state]; the initial one is 0 if None. Returns y, or
    (y, final_state). Differentiable once, in every tensor but the offsets; gradients are the same from run to run.
    """
    require_cuda(x, dt, A, B, C, D, z, dt_bias, initial_state, seq_offsets)
    n_seq, _, _ = check_offsets(seq_offsets, x)
    B, C, dim, state, _ = _check(x, dt, A, B, C, D, z, dt_bias)
    if initial_state is not None:
        check_shape("initial_state", initial_state, (n_seq, dim, state))
        check_dtype("initial_state", initial_state, torch.float32)
        initial_state = dense(initial_state)
    args = (x, dt, _float(A), B, C, _float(D), z, _float(dt_bias), initial_state, seq_offsets, bool(dt_softplus),
            bool(return_final_state))
    if needs_grad(x, dt, A, B, C, D, z, dt_bias, initial_state):
        y, final = _SelectiveScan.apply(*args)
    else:
        y, final = _forward(*args, False)[:2]
    return (y, final) if return_final_state else y


def selective_scan_update(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                          state: torch.Tensor, D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None,
                          dt_bias: Optional[torch.Tensor] = None, dt_softplus: bool = True,
                          state_indices: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One more token: x, dt, z [rows, dim], B, C [rows, state] or [rows, groups, state] -> y [rows, dim].

    ``state`` [slots, dim, state] fp32 is updated in place. Row i uses slot ``state_indices[i]`` (int32 on the
    device, distinct), or slot i without indices; a row whose index is no slot is padding: its y is 0 and no state
    changes. Up to 262140 rows. Not differentiable: where an input asks for a gradient, a backward pass through y
    raises.
    """
    require_cuda(x, dt, A, B, C, state, D, z, dt_bias, state_indices)
    if torch.is_grad_enabled() and (x.requires_grad or dt.requires_grad or A.requires_grad or B.requires_grad
                                    or C.requires_grad or state.requires_grad
                                    or (D is not None and D.requires_grad) or (z is not None and z.requires_grad)
                                    or (dt_bias is not None and dt_bias.requires_grad)):
        return without_gradient(selective_scan_update, x, dt, A, B, C, state, D, z, dt_bias, dt_softplus,
                                state_indices)
    key = (x.shape, x.stride(), x.dtype, dt.shape, dt.stride(), dt.dtype, B.shape, B.stride(), B.dtype, C.shape,
           C.stride(), C.dtype, A.shape, A.stride(), A.dtype, state.shape, state.stride(), state.dtype,
           None if D is None else (D.shape, D.stride(), D.dtype), None if z is None else (z.shape, z.stride(), z.dtype),
           layout(dt_bias), layout(state_indices), dt_softplus)
    desc = _update_plans.get(key)
    if desc is None:
        x, dt, A, B, C, D, z, dt_bias, desc = _update_plan(x, dt, A, B, C, state, D, z, dt_bias, dt_softplus,
                                                           state_indices, key)
    y = x.new_empty(x.shape)
    call_on(x.get_device(), "sf_selective_scan_update", x.data_ptr(), dt.data_ptr(), A.data_ptr(), B.data_ptr(),
            C.data_ptr(), ptr(D), ptr(z), ptr(dt_bias), state.data_ptr(), ptr(state_indices), y.data_ptr(),
            state.shape[0], desc)
    written((state,))
    return y


# Descriptors of the layouts that single-token calls have come with, where nothing had to be copied: a decoding loop's
# next call with the same layouts has passed its checks.
_update_plans: dict = {}


def _update_plan(x, dt, A, B, C, state, D, z, dt_bias, dt_softplus, state_indices, key):
    """Checks a call and returns its operands as the kernel reads them and its descriptor."""
    if x.dim() != 2:
        raise ValueError(f"x: expected [rows, dim], got {list(x.shape)}")
    given = (x, dt, A, B, C, D, z, dt_bias)
    B, C, dim, n, groups = _check(x, dt, A, B, C, D, z, dt_bias)
    if state.dim() != 3 or not state.is_contiguous():
        raise ValueError("state: expected a contiguous [slots, dim, state] tensor")
    check_shape("state", state, (state.shape[0], dim, n))
    check_dtype("state", state, torch.float32)
    check_state_indices(state_indices, x.shape[0], state.shape[0])
    A, D, dt_bias = _float(A), _float(D), _float(dt_bias)
    x, dt, z, B, C, strides = _strided(x, dt, z, B, C)
    desc = _lib.selective_scan_desc(1, strides, x.shape[0], dim, n, groups, bool(dt_softplus), x.dtype, False)
    args = (x, dt, A, B, C, D, z, dt_bias)
    if all(a is b or (a is not None and a.data_ptr() == b.data_ptr() and a.dtype is b.dtype)
           for a, b in zip(args, given)):
        if len(_update_plans) >= 512:
            _update_plans.clear()
        _update_plans[key] = desc
    return (*args, desc)
