"""The norms around a block with its gate and residual scale, in one kernel (csrc/block_norm.cu).

No counterpart in the reference (its blocks normalise by batch statistics, folded into convolutions).
"""
from __future__ import annotations

from typing import Optional

import torch

from .. import _lib
from ._sequence import call_on, check_dtype, check_shape, dense, layout, needs_grad, ptr, require_cuda

_GATES = {None: _lib.SF_GATE_LINEAR, "silu": _lib.SF_GATE_SILU, "sigmoid": _lib.SF_GATE_SIGMOID}
_MAX_DIM = 16384


def _rows(t: Optional[torch.Tensor], dim: int):
    """t as rows of contiguous channels (a copy only where they are not evenly spaced) and its row stride."""
    if t is None:
        return None, 0
    if t.is_contiguous():
        return t, dim
    t = t.reshape(-1, dim)
    if dim != 1 and t.stride(1) != 1:
        t = t.contiguous()
    return t, t.stride(0) if t.shape[0] > 1 else dim


def _empty(shape, dtype, device):
    return torch.empty(shape, dtype=dtype, device=device)


def _forward(y, residual, gate, post_weight, pre_weight, scale, rows_per_gate, kind, residual_scale, eps, res_dtype,
             want_rstd):
    shape, dim = y.shape, y.shape[-1]
    w = post_weight if post_weight is not None else pre_weight if pre_weight is not None else scale
    y, y_row = _rows(y, dim)
    residual, r_row = _rows(residual, dim)
    gate, g_row = _rows(gate, dim)
    rows = y.numel() // dim
    desc = _lib.block_norm_desc(rows, y_row, r_row, g_row, rows_per_gate, dim, y.dtype, res_dtype,
                                y.dtype if w is None else w.dtype, kind, residual_scale, eps)
    r_out = y.new_empty(shape, dtype=res_dtype)
    x_out = None if pre_weight is None else y.new_empty(shape)
    rstd = y.new_empty(2 * rows, dtype=torch.float32) if want_rstd else None
    call_on(y.get_device(), "sf_block_norm", ptr(y), ptr(residual), ptr(gate), ptr(post_weight), ptr(pre_weight), ptr(scale),
            ptr(r_out), ptr(x_out), ptr(rstd), desc)
    return r_out, x_out, rstd, desc, (y, residual, gate)


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, residual, gate, post_weight, pre_weight, scale, *rest):
        ctx.shapes = tuple(None if t is None else t.shape for t in (y, residual, gate))
        r_out, x_out, rstd, ctx.desc, (y, residual, gate) = _forward(y, residual, gate, post_weight, pre_weight, scale,
                                                                     *rest, True)
        ctx.save_for_backward(y, residual, gate, post_weight, pre_weight, scale, rstd)
        ctx.set_materialize_grads(False)
        return r_out, x_out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dr, dx):
        y, residual, gate, post_weight, pre_weight, scale, rstd = ctx.saved_tensors

        def like(t):
            return None if t is None else t.new_empty(t.shape)

        dr = dense(dr)
        dx = dense(dx)
        dy, dres, dgate, dpost, dpre, dscale = (like(t) for t in (y, residual, gate, post_weight, pre_weight, scale))
        if dgate is not None and not y.numel():  # gates of sequences without rows, which no kernel meets
            dgate.zero_()
        nbytes = _lib.load().sf_block_norm_backward_workspace_size(ctx.desc)
        ws = _empty(max(nbytes, 1), torch.uint8, y.device)
        call_on(y.get_device(), "sf_block_norm_backward", ptr(y), ptr(residual), ptr(gate), ptr(post_weight), ptr(pre_weight),
                ptr(scale), ptr(rstd), ptr(dr), ptr(dx), ptr(dy), ptr(dres), ptr(dgate), ptr(dpost), ptr(dpre),
                ptr(dscale), ctx.desc, ptr(ws), nbytes)
        grads = [None if g is None else g.view(s) for g, s in zip((dy, dres, dgate), ctx.shapes)]
        return (*grads, dpost, dpre, dscale, None, None, None, None, None)


def block_norm(y: torch.Tensor, residual: Optional[torch.Tensor] = None, post_weight: Optional[torch.Tensor] = None,
               pre_weight: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
               gate_activation: Optional[str] = None, scale: Optional[torch.Tensor] = None,
               residual_scale: float = 1.0, eps: float = 1e-6, residual_dtype: Optional[torch.dtype] = None):
    """What stands between two blocks: (residual_out, normed) with

        residual_out = residual_scale * residual + scale * act(gate) * (post_weight * y / rms(y))
        normed = pre_weight * residual_out / rms(residual_out),   rms(v) = sqrt(mean(v^2) + eps)

    y [..., dim] (dim up to 16384) is the block's output. Every other part may be left out: no ``post_weight``: y
    itself; no ``residual``: 0, and residual_out is of ``residual_dtype`` (y's type if None); no ``pre_weight``: no
    second norm, normed is None. ``gate`` has y's type and shape, or 1 for the second last dimension (one gate row
    for the rows of a sequence); ``gate_activation`` None, "silu" or "sigmoid". ``scale`` and the weights [dim] are
    of one type, y's or fp32; the residual is of y's type or fp32, and its rounding does not enter ``normed``.
    Differentiable once, in every tensor.
    """
    require_cuda(y, residual, post_weight, pre_weight, gate, scale)
    if needs_grad(y, residual, gate, post_weight, pre_weight, scale):
        return _BlockNorm.apply(*_check(y, residual, post_weight, pre_weight, gate, gate_activation, scale, residual_scale,
                                        eps, residual_dtype))
    key = (layout(y), layout(residual), layout(post_weight), layout(pre_weight), layout(gate), gate_activation,
           layout(scale), residual_scale, eps, residual_dtype)
    plan = _plans.get(key)
    if plan is None:
        args = _check(y, residual, post_weight, pre_weight, gate, gate_activation, scale, residual_scale, eps,
                      residual_dtype)
        r_out, x_out, _, desc, _ = _forward(*args, False)
        if all(t is None or t.is_contiguous() for t in (y, residual, post_weight, pre_weight, gate, scale)):
            if len(_plans) >= 512:
                _plans.clear()
            _plans[key] = (desc, args[-1])
        return r_out, x_out
    desc, res_dtype = plan
    r_out = y.new_empty(y.shape, dtype=res_dtype)
    x_out = None if pre_weight is None else y.new_empty(y.shape)
    call_on(y.get_device(), "sf_block_norm", y.data_ptr(), ptr(residual), ptr(gate), ptr(post_weight), ptr(pre_weight),
            ptr(scale), r_out.data_ptr(), ptr(x_out), None, desc)
    return r_out, x_out


# Descriptors of the layouts that calls without gradients have come with, where all tensors are contiguous: a decoding
# loop's next call with the same layouts has passed its checks.
_plans: dict = {}


def _check(y, residual, post_weight, pre_weight, gate, gate_activation, scale, residual_scale, eps, residual_dtype):
    """Checks a call and returns the arguments of _forward."""
    _lib.sf_dtype(y.dtype)
    if y.dim() < 1 or not 1 <= y.shape[-1] <= _MAX_DIM:
        raise ValueError(f"y: expected [..., dim] with dim up to {_MAX_DIM}, got {list(y.shape)}")
    dim = y.shape[-1]
    if gate_activation not in _GATES:
        raise ValueError(f"gate_activation: expected None, 'silu' or 'sigmoid', got {gate_activation!r}")
    w_dtype = None
    for name, t in (("post_weight", post_weight), ("pre_weight", pre_weight), ("scale", scale)):
        if t is None:
            continue
        check_shape(name, t, (dim,))
        w_dtype = t.dtype if w_dtype is None else w_dtype
        check_dtype(name, t, w_dtype)
        if t.dtype not in (y.dtype, torch.float32):
            raise TypeError(f"{name}: expected {y.dtype} or torch.float32, got {t.dtype}")
    if residual is not None:
        check_shape("residual", residual, y.shape)
        if residual_dtype not in (None, residual.dtype):
            raise TypeError(f"residual_dtype is {residual_dtype}, the residual {residual.dtype}")
        residual_dtype = residual.dtype
    residual_dtype = residual_dtype or y.dtype
    if residual_dtype not in (y.dtype, torch.float32):
        raise TypeError(f"residual: expected {y.dtype} or torch.float32, got {residual_dtype}")
    rows_per_gate = 1
    if gate is not None:
        check_dtype("gate", gate, y.dtype)
        if gate.shape != y.shape:
            if y.dim() < 2 or tuple(gate.shape) != (*y.shape[:-2], 1, dim):
                raise ValueError(f"gate: expected {list(y.shape)} or {[*y.shape[:-2], 1, dim]}, got {list(gate.shape)}")
            rows_per_gate = max(1, y.shape[-2])
    post_weight, pre_weight, scale = dense(post_weight), dense(pre_weight), dense(scale)
    return (y, residual, gate, post_weight, pre_weight, scale, rows_per_gate,
            _lib.SF_GATE_NONE if gate is None else _GATES[gate_activation], float(residual_scale), float(eps),
            residual_dtype)
