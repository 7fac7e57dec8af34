"""The 64-bit formulas that the GPU tests compare against, checked by differences; refusals that need no GPU."""
import pytest
import torch

import sequence_reference as ref


def _check(fn, inputs, grads, eps=1e-6):
    """Every gradient of sum(fn(inputs)) by central differences along a random direction of each input."""
    g = torch.Generator().manual_seed(5)
    for name, t in inputs.items():
        v = torch.randn(t.shape, generator=g, dtype=torch.float64)
        up, down = (fn(**{**inputs, name: t + s * eps * v}) for s in (1, -1))
        diff = float((up - down) / (2 * eps))
        want = float((grads[name] * v).sum())
        # Truncation eps^2 and rounding 1e-16 / eps of a loss of order 10 to 100.
        assert abs(diff - want) <= 1e-7 * (1 + abs(want)) * 10, (name, diff, want)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, dtype=torch.float64)


@pytest.mark.parametrize("act", [False, True])
@pytest.mark.parametrize("lengths", [[5, 0, 1, 7], [2, 3]])
def test_conv_gradients_by_differences(act, lengths):
    g = torch.Generator().manual_seed(1)
    n, dim, w = sum(lengths), 3, 4
    offsets = [0] + torch.tensor(lengths).cumsum(0).tolist()
    inp = {"x": _normal(g, n, dim), "weight": _normal(g, dim, w), "bias": _normal(g, dim),
           "init": _normal(g, len(lengths), w - 1, dim)}
    dy, df = _normal(g, n, dim), _normal(g, len(lengths), w - 1, dim)

    def loss(x, weight, bias, init):
        y, f = ref.conv(x, weight, bias, act, init, offsets)[:2]
        return (y * dy).sum() + (f * df).sum()

    _, _, dx, dw, db, di = ref.conv(inp["x"], inp["weight"], inp["bias"], act, inp["init"], offsets, dy, df)
    _check(loss, inp, {"x": dx, "weight": dw, "bias": db, "init": di})


@pytest.mark.parametrize("softplus", [False, True])
@pytest.mark.parametrize("gated", [False, True])
def test_scan_gradients_by_differences(softplus, gated):
    g = torch.Generator().manual_seed(2)
    lengths, dim, n, groups = [4, 0, 1, 6], 4, 3, 2
    total, offsets = sum(lengths), [0] + torch.tensor(lengths).cumsum(0).tolist()
    inp = {"x": _normal(g, total, dim), "dt": _normal(g, total, dim).abs(), "A": -_normal(g, dim, n).abs(),
           "B": _normal(g, total, groups, n), "C": _normal(g, total, groups, n), "D": _normal(g, dim),
           "bias": 0.1 * _normal(g, dim), "init": _normal(g, len(lengths), dim, n)}
    if gated:
        inp["z"] = _normal(g, total, dim)
    dy, df = _normal(g, total, dim), _normal(g, len(lengths), dim, n)

    def loss(x, dt, A, B, C, D, bias, init, z=None):
        o = ref.scan(x, dt, A, B, C, D, z, bias, softplus, init, offsets)
        return (o["y"] * dy).sum() + (o["final"] * df).sum()

    o = ref.scan(inp["x"], inp["dt"], inp["A"], inp["B"], inp["C"], inp["D"], inp.get("z"), inp["bias"], softplus,
                 inp["init"], offsets, dy, df)
    _check(loss, inp, {k: o["d" + k] for k in inp})


@pytest.mark.parametrize("kind", [None, "linear", "silu", "sigmoid"])
@pytest.mark.parametrize("post, pre", [(True, True), (False, True), (True, False)])
def test_norm_gradients_by_differences(kind, post, pre):
    g = torch.Generator().manual_seed(3)
    shape = (2, 3, 5)
    inp = {"y": _normal(g, *shape), "residual": _normal(g, *shape), "scale": _normal(g, 5)}
    if kind:
        inp["gate"] = _normal(g, 2, 1, 5)
    if post:
        inp["w_post"] = _normal(g, 5)
    if pre:
        inp["w_pre"] = _normal(g, 5)
    dr, dx = _normal(g, *shape), _normal(g, *shape)

    def run(y, residual, scale, gate=None, w_post=None, w_pre=None, **kw):
        return ref.norm(y, residual, gate, kind, w_post, w_pre, scale, 0.7, 1e-3, **kw)

    def loss(**kw):
        o = run(**kw)
        return (o["r"] * dr).sum() + ((o["x"] * dx).sum() if pre else 0)

    o = run(**inp, dr=dr, dx=dx if pre else None)
    names = {"y": "dy", "residual": "dres", "scale": "dscale", "gate": "dgate", "w_post": "dpost", "w_pre": "dpre"}
    _check(loss, inp, {k: o[names[k]] for k in inp})


def test_cpu_tensors_are_refused():
    from sparseflow_b200.Kernels.block_norm import block_norm
    from sparseflow_b200.Kernels.causal_conv1d import causal_conv1d, causal_conv1d_update
    from sparseflow_b200.Kernels.selective_scan import selective_scan, selective_scan_update
    x, w, A, b = torch.zeros(1, 2, 4), torch.zeros(4, 3), torch.zeros(4, 2), torch.zeros(1, 2, 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        causal_conv1d(x, w)
    with pytest.raises(RuntimeError, match="CUDA"):
        causal_conv1d_update(x[0], torch.zeros(2, 2, 4), w)
    with pytest.raises(RuntimeError, match="CUDA"):
        selective_scan(x, x, A, b, b)
    with pytest.raises(RuntimeError, match="CUDA"):
        selective_scan_update(x[0], x[0], A, b[0], b[0], torch.zeros(2, 4, 2))
    with pytest.raises(RuntimeError, match="CUDA"):
        block_norm(x)
