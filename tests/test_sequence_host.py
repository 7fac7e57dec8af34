"""The host side of the sequence operators, without a GPU."""
import ctypes
import itertools
import subprocess
import sys
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parent.parent


def _in_a_process(code):
    """Runs code that would end the process where the host arithmetic faults."""
    r = subprocess.run([sys.executable, "-c", "import ctypes, itertools\nfrom sparseflow_b200 import _lib\nlib = _lib.load()\n" + code],
                       cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0, (r.returncode, r.stderr[-500:])


def test_block_norm_workspace_of_any_shape():
    """Every count of rows, rows per gate and channels has a workspace size, what the entries refuse has 0; none divides
    by zero."""
    _in_a_process("""
for rows, per, dim, gate in itertools.product((0, 1, 6, 1 << 40), (1, 2, 6), (1, 7, 4096, 16384, 20000, 1 << 30), (0, 2)):
    d = _lib.BlockNormDesc(rows, dim, dim, dim, per, dim, 0, 0, 0, gate, 1.0, 1e-6)
    n = lib.sf_block_norm_backward_workspace_size(ctypes.byref(d))
    assert (n > 0) == (rows % per == 0 and dim <= 16384), (rows, per, dim, gate, n)
""")


def test_selective_scan_workspace_of_any_shape():
    """Sizes of every shape that the entries take, and 0 for states that they refuse."""
    _in_a_process("""
for length, n, dim, state, groups, packed in itertools.product((0, 1, 17, 1 << 33), (0, 1, 3), (0, 8, 1 << 20),
                                                               (1, 16, 128, 129, 1025, 5000, 2 ** 31 - 1), (1, 8), (0, 1)):
    d = ctypes.byref(_lib.SelectiveScanDesc(length, *[0] * 10, n, dim, state, groups, 1, 0, packed))
    sizes = [lib.sf_selective_scan_checkpoint_bytes(d), lib.sf_selective_scan_workspace_size(d),
             lib.sf_selective_scan_backward_workspace_size(d)]
    assert state <= 128 or not any(sizes), sizes
    assert state > 128 or n == 0 or dim == 0 or (sizes[0] > 0 and sizes[2] > 0), sizes
""")


@pytest.mark.parametrize("inner", [1, 2])
@pytest.mark.parametrize("empty", [lambda t: t.transpose(1, 3)[:, :0], lambda t: t.transpose(1, 3)[:0],
                                   lambda t: t[:, :0].permute(0, 3, 2, 1), lambda t: t.permute(3, 2, 1, 0)[..., :0]])
def test_rows_of_empty_views(empty, inner):
    """Views without elements in any order of dimensions: strides of a contiguous tensor, and no endless recursion."""
    from sparseflow_b200.Kernels._sequence import rows_of
    t = empty(torch.zeros(2, 8, 5, 7))
    got, batch, row = rows_of(t, inner)
    assert got.shape == t.shape and row >= 0 and batch >= 0


def test_spiking_steps_refuse_slots_and_other_rows():
    """The membranes of a spiking mixer go by row: a pool's slots, or another number of rows, would mix requests."""
    from sparseflow_b200.Ops.state_space import StateSpaceMixer
    m = StateSpaceMixer(8, spiking=True).eval()
    state = m.new_state(4)
    before = [s.clone() for s in state]
    with pytest.raises(ValueError, match="spiking"):
        m.step(torch.zeros(2, 8), state, torch.tensor([3, 0], dtype=torch.int32))
    m.lif.v = torch.zeros(4, m.inner)
    with pytest.raises(ValueError, match="reset_net"):
        m.step(torch.zeros(2, 8), state)
    assert all(torch.equal(a, b) for a, b in zip(state, before))


def _calls():
    """A call of each operator on CPU tensors, by the names of its tensors."""
    from sparseflow_b200.Kernels.block_norm import block_norm
    from sparseflow_b200.Kernels.causal_conv1d import causal_conv1d, causal_conv1d_update
    from sparseflow_b200.Kernels.selective_scan import selective_scan, selective_scan_update
    x, w, A, b = torch.ones(1, 2, 4), torch.ones(4, 3), -torch.ones(4, 2), torch.ones(1, 2, 2)
    return [(causal_conv1d, dict(x=x, weight=w, bias=w[:, 0], initial_state=torch.ones(1, 2, 4))),
            (causal_conv1d_update, dict(x=x[0], state=torch.ones(2, 2, 4), weight=w, bias=w[:, 0])),
            (selective_scan, dict(x=x, dt=x, A=A, B=b, C=b, D=w[:, 0], z=x, dt_bias=w[:, 0],
                                  initial_state=torch.ones(1, 4, 2))),
            (selective_scan_update, dict(x=x[0], dt=x[0], A=A, B=b[0], C=b[0], state=torch.ones(2, 4, 2), D=w[:, 0],
                                         z=x[0], dt_bias=w[:, 0])),
            (block_norm, dict(y=x, residual=x, post_weight=w[:, 0], pre_weight=w[:, 0], gate=x, scale=w[:, 0]))]


@pytest.mark.parametrize("which", range(5))
def test_tangents_are_refused(which):
    """No operator has a forward-mode derivative: a dual tensor in any place raises, and plain ones do not."""
    fn, tensors = _calls()[which]
    with torch.autograd.forward_ad.dual_level():
        for name, t in tensors.items():
            dual = torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                fn(**{**tensors, name: dual})
        with pytest.raises(RuntimeError, match="CUDA"):
            fn(**tensors)


@pytest.mark.parametrize("cast", [lambda m: m.bfloat16(), lambda m: m.half(), lambda m: m.to(torch.bfloat16),
                                  lambda m: m.to("cpu", torch.float16)])
def test_scan_parameters_stay_in_32_bits(cast):
    """Casting a model leaves the parameters that the scan reads in 32 bits as they are, and their gradients."""
    from sparseflow_b200.snn import SpikingStateSpaceLM
    m = SpikingStateSpaceLM(10, 16, 2)
    m.mixers[0].D.grad = torch.full_like(m.mixers[0].D, 1.001)
    before = [(p.A_log.clone(), p.dt_bias.clone(), p.D.clone()) for p in m.mixers]
    cast(m)
    for mixer, want in zip(m.mixers, before):
        for got, value in zip((mixer.A_log, mixer.dt_bias, mixer.D), want):
            assert isinstance(got, torch.nn.Parameter) and got.dtype == torch.float32 and torch.equal(got, value)
        assert mixer.in_proj.weight.dtype == mixer.conv_weight.dtype == m.embedding.weight.dtype != torch.float32
    assert m.mixers[0].D.grad.dtype == torch.float32 and (m.mixers[0].D.grad == torch.tensor(1.001)).all()
    m.float()
    assert all(p.dtype == torch.float32 for p in m.parameters())
    assert m.to("meta").mixers[1].A_log.is_meta
