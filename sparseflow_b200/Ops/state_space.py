"""Layers of a spiking language model around the selective state space scan.

``StateSpaceMixer`` is to a sequence of tokens what a convolution with its LIF neuron is to frames: a short causal
convolution, the selective scan (the learned, linear counterpart of the membrane), and, where it spikes, a
``LIFNode`` over the tokens whose spikes drive an event-driven ``SparseLinear``. ``BlockNorm`` stands between blocks.
No counterpart in the reference.
"""
from __future__ import annotations

import math
from typing import Optional

import torch
import torch.nn as nn

from ..Kernels.block_norm import block_norm
from ..Kernels.causal_conv1d import causal_conv1d, causal_conv1d_update
from ..Kernels.selective_scan import selective_scan, selective_scan_update
from .lif_node import LIFNode
from .sparse_linear import SparseLinear


class StateSpaceMixer(nn.Module):
    """[batch, length, dim] -> [batch, length, dim]: projection to 2 x inner channels (x and its gate z), short causal
    convolution with SiLU, selective scan, projection back.

    ``spiking``: the scan's output passes a LIF neuron over the tokens and the projection back is a ``SparseLinear`` of
    its spikes (the membrane is kept between calls like any ``LIFNode``'s, see ``reset_net``). Without it the
    projection is dense and the layer is differentiable; the LIF neuron and the SparseLinear are inference operators.
    ``A_log``, ``dt_bias`` and ``D`` stay fp32 when the layer is cast to another type: 16 bits would hold a step of 1e-3,
    whose bias is near -6.9, to 1.6 %, and the scan reads them in 32 bits.
    """

    def __init__(self, dim: int, state: int = 16, width: int = 4, expand: int = 2, dt_rank: Optional[int] = None,
                 groups: int = 1, spiking: bool = False, tau: float = 2.0, v_threshold: float = 1.0):
        super().__init__()
        self.inner = inner = expand * dim
        self.state, self.groups = state, groups
        self.dt_rank = dt_rank or max(1, dim // 16)
        self.in_proj = nn.Linear(dim, 2 * inner, bias=False)
        self.conv_weight = nn.Parameter(torch.empty(inner, width).uniform_(-1, 1) / math.sqrt(width))
        self.conv_bias = nn.Parameter(torch.zeros(inner))
        self.x_proj = nn.Linear(inner, self.dt_rank + 2 * groups * state, bias=False)
        self.dt_proj = nn.Linear(self.dt_rank, inner, bias=False)
        # Steps of 1e-3 to 1e-1, spread over the logarithm; dt_bias is their inverse softplus.
        step = torch.exp(torch.rand(inner) * math.log(100.0) + math.log(1e-3))
        self.dt_bias = nn.Parameter(step + torch.log(-torch.expm1(-step)))
        self.A_log = nn.Parameter(torch.log(torch.arange(1, state + 1, dtype=torch.float32)).repeat(inner, 1))
        self.D = nn.Parameter(torch.ones(inner))
        self.lif = LIFNode(tau=tau, v_threshold=v_threshold) if spiking else None
        self.out_proj = SparseLinear(inner, dim) if spiking else nn.Linear(inner, dim)

    def _apply(self, fn, recurse=True):
        fp32 = [t for p in (self.A_log, self.dt_bias, self.D) for t in (p, p.grad) if t is not None]

        def keep(t):
            out = fn(t)
            return t.to(out.device) if out.dtype != t.dtype and any(t is p for p in fp32) else out
        return super()._apply(keep, recurse)

    def new_state(self, batch: int):
        """(convolution state, scan state) of `batch` sequences that have not begun."""
        w = self.conv_weight
        return (torch.zeros(batch, w.shape[1] - 1, self.inner, dtype=w.dtype, device=w.device),
                torch.zeros(batch, self.inner, self.state, dtype=torch.float32, device=w.device))

    def _selection(self, x):
        """dt, B and C of the convolution's output; B and C are slices of the projection's rows."""
        p = self.x_proj(x)
        n = self.groups * self.state
        B, C = (p[..., self.dt_rank + i * n: self.dt_rank + (i + 1) * n].unflatten(-1, (self.groups, self.state))
                for i in (0, 1))
        return self.dt_proj(p[..., : self.dt_rank]), B, C

    def _A(self):
        return -torch.exp(self.A_log.float())

    def forward(self, u: torch.Tensor, seq_offsets: Optional[torch.Tensor] = None, state=None):
        """u [batch, length, dim], or [total, dim] of packed sequences (not if spiking). Returns the output, or with
        ``state`` (from ``new_state`` or an earlier call) (output, state after it)."""
        if self.lif is not None and seq_offsets is not None:
            raise ValueError("packed sequences need spiking=False: the LIF neuron runs over equally long sequences")
        if self.lif is not None and self.training and torch.is_grad_enabled():
            raise RuntimeError("a spiking mixer has no gradient: train with spiking=False, or call eval() / no_grad()")
        x, z = self.in_proj(u).split(self.inner, -1)
        x = causal_conv1d(x, self.conv_weight, self.conv_bias, "silu", None if state is None else state[0], seq_offsets,
                          state is not None)
        if state is not None:
            x, conv_state = x
        dt, B, C = self._selection(x)
        y = selective_scan(x, dt, self._A(), B, C, self.D, z, self.dt_bias,
                           initial_state=None if state is None else state[1], seq_offsets=seq_offsets,
                           return_final_state=state is not None)
        if state is not None:
            y, scan_state = y
        if self.lif is not None:
            y = self.lif(y.transpose(0, 1)).transpose(0, 1)
        out = self.out_proj(y)
        return out if state is None else (out, (conv_state, scan_state))

    def step(self, u: torch.Tensor, state, state_indices: Optional[torch.Tensor] = None) -> torch.Tensor:
        """One token for each row of u [rows, dim]; the states (pools, where indices are given) are updated in place.
        A spiking mixer takes the same rows in the same order at every step, as its membranes go by row."""
        if self.lif is not None:
            if state_indices is not None:
                raise ValueError("state_indices need spiking=False: the LIF neuron's membranes go by row, not by slot")
            if self.lif.v is not None and self.lif.v.shape[0] != u.shape[0]:
                raise ValueError(f"{u.shape[0]} rows, but membranes of {self.lif.v.shape[0]}: reset_net() before "
                                 "another batch")
        x, z = self.in_proj(u).split(self.inner, -1)
        x = causal_conv1d_update(x, state[0], self.conv_weight, self.conv_bias, "silu", state_indices)
        dt, B, C = self._selection(x)
        y = selective_scan_update(x, dt, self._A(), B, C, state[1], self.D, z, self.dt_bias,
                                  state_indices=state_indices)
        if self.lif is not None:
            y = self.lif(y[None])[0]
        return self.out_proj(y)


class BlockNorm(nn.Module):
    """The norm after a block, its gate and layer scale, the residual, and the norm before the next block, as one
    ``block_norm`` call: (block output, residual, gate) -> (residual, normed)."""

    def __init__(self, dim: int, scale: float = 1.0, gate_activation: Optional[str] = "silu", eps: float = 1e-6):
        super().__init__()
        self.post_weight = nn.Parameter(torch.ones(dim))
        self.pre_weight = nn.Parameter(torch.ones(dim))
        self.scale = nn.Parameter(torch.full((dim,), float(scale)))
        self.gate_activation, self.eps = gate_activation, eps

    def forward(self, y, residual, gate=None):
        return block_norm(y, residual, self.post_weight, self.pre_weight, gate=gate,
                          gate_activation=self.gate_activation, scale=self.scale, eps=self.eps)
