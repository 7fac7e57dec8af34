"""block_norm against the formulas in 64 bits."""
import pytest
import torch

import sequence_reference as ref

pytestmark = pytest.mark.gpu

# fp32 roundings: a tree of sums over a row (at most 16 in a thread and 10 levels), the root, the activation, products.
FWD = 64
TYPES = [torch.float32, torch.float16, torch.bfloat16]
KINDS = {"linear": None, "silu": "silu", "sigmoid": "sigmoid"}


def _make(dtype, shape, res=None, wdtype=torch.float32, gate="rows", post=True, pre=True, scale=True, residual=True):
    g = torch.Generator(device="cuda").manual_seed(7)

    def r(*s, dt=dtype):
        return torch.randn(*s, device="cuda", generator=g).to(dt)
    dim, res = shape[-1], res or dtype
    gshape = {"rows": shape, "sequence": (*shape[:-2], 1, dim)}.get(gate)
    return dict(y=r(*shape), residual=r(*shape, dt=res) if residual else None, gate=r(*gshape) if gshape else None,
                post=r(dim, dt=wdtype) if post else None, pre=r(dim, dt=wdtype) if pre else None,
                scale=r(dim, dt=wdtype) if scale else None, dr=r(*shape, dt=res), dx=r(*shape))


def _call(m, kind="silu", **kw):
    from sparseflow_b200.Kernels.block_norm import block_norm
    return block_norm(m["y"], m["residual"], m["post"], m["pre"], gate=m["gate"], gate_activation=KINDS[kind],
                      scale=m["scale"], residual_scale=0.75, eps=1e-5, **kw)


def _run_and_compare(m, kind="silu", use=("dr", "dx")):
    names = [k for k in ("y", "residual", "gate", "post", "pre", "scale") if m[k] is not None]
    leaves = {k: m[k].detach().requires_grad_() for k in names}
    r, x = _call({**m, **leaves}, kind)
    r2, x2 = _call(m, kind)
    assert torch.equal(r, r2) and (x is None) == (x2 is None) and (x is None or torch.equal(x, x2))
    use = [k for k in use if k == "dr" or x is not None]
    grads = dict(zip(names, torch.autograd.grad([{"dr": r, "dx": x}[k] for k in use], list(leaves.values()),
                                                [m[k] for k in use], allow_unused=True)))
    y, res, gate, post, pre, scale = ref.f64(*(m[k] for k in ("y", "residual", "gate", "post", "pre", "scale")))
    args = (y, res, gate, kind if gate is not None else None, post, pre, scale, 0.75, 1e-5)
    kw = {k: ref.f64(m[k]) for k in use}
    val, mag = ref.norm(*args, **kw), ref.norm(*args, **kw, mag=True)
    ref.close(r, val["r"], mag["r"], FWD, "residual")
    if x is not None:
        ref.close(x, val["x"], mag["x"], FWD, "normed")
    rows = y.numel() // y.shape[-1]
    for k, n in (("y", "dy"), ("residual", "dres"), ("gate", "dgate"), ("post", "dpost"), ("pre", "dpre"),
                 ("scale", "dscale")):
        if k in names:
            ref.close(grads[k], val[n], mag[n], 4 * FWD + (rows if k not in ("y", "residual") else 0), k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [1, 7, 64, 257, 1000, 2048, 4104, 8200, 16384])
@pytest.mark.parametrize("gate", ["rows", "sequence", None])
def test_widths_and_gates(dtype, dim, gate):
    _run_and_compare(_make(dtype, (2, 3, dim), gate=gate))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("wide", [False, True])
def test_activations_and_types(dtype, kind, wide):
    f32 = torch.float32
    _run_and_compare(_make(dtype, (3, 11, 96), res=f32 if wide else dtype, wdtype=f32 if wide else dtype), kind)


@pytest.mark.parametrize("left_out", [("post",), ("pre",), ("scale",), ("residual",), ("post", "scale"),
                                      ("pre", "residual"), ("post", "pre", "scale")])
@pytest.mark.parametrize("gate", ["rows", None])
def test_parts_left_out(left_out, gate):
    _run_and_compare(_make(torch.bfloat16, (5, 4, 136), gate=gate, **{k: False for k in left_out}))


@pytest.mark.parametrize("use", [("dr",), ("dx",)])
def test_gradient_of_one_output(use):
    _run_and_compare(_make(torch.float32, (2, 9, 72)), use=use)


@pytest.mark.parametrize("shape", [(1, 1, 64), (1, 2000, 64), (37, 50, 40), (700, 1, 48)])
@pytest.mark.parametrize("gate", ["rows", "sequence"])
def test_many_rows(shape, gate):
    """More rows than blocks; blocks that hold parts of sequences."""
    _run_and_compare(_make(torch.bfloat16, shape, gate=gate, res=torch.float32))


def test_rows_of_zeros():
    m = _make(torch.float32, (2, 4, 64))
    m["y"][0, 1] = 0
    m["residual"][0, 1] = 0
    _run_and_compare(m)


def test_first_norm_of_a_model():
    """Without a block before: y enters the residual stream in fp32 as it is."""
    from sparseflow_b200.Kernels.block_norm import block_norm
    y, w = torch.randn(3, 5, 64, device="cuda").bfloat16(), torch.randn(64, device="cuda")
    r, x = block_norm(y, pre_weight=w, residual_dtype=torch.float32)
    assert r.dtype == torch.float32 and torch.equal(r, y.float())
    val = ref.norm(ref.f64(y), None, None, None, None, ref.f64(w), None, 1.0, 1e-6)
    mag = ref.norm(ref.f64(y), None, None, None, None, ref.f64(w), None, 1.0, 1e-6, mag=True)
    ref.close(x, val["x"], mag["x"], FWD)


@pytest.mark.parametrize("offset, pad", [(0, 8), (8, 16), (3, 2)])
def test_slices_of_wider_rows(offset, pad):
    m = _make(torch.bfloat16, (4, 6, 64))
    w = dict(m)
    for k in ("y", "gate", "residual"):
        wide = torch.full((4, 6, offset + 64 + pad), 3.0, device="cuda", dtype=m[k].dtype)
        wide[..., offset:offset + 64] = m[k]
        w[k] = wide[..., offset:offset + 64]
    for a, b in zip(_call(w), _call(m)):
        assert torch.equal(a, b)
    w["y"] = m["y"].transpose(0, 1).contiguous().transpose(0, 1)
    w["gate"] = m["gate"].transpose(1, 2).contiguous().transpose(1, 2)
    w["residual"] = m["residual"][:1].expand(4, 6, 64)
    m["residual"] = w["residual"].contiguous()
    for a, b in zip(_call(w), _call(m)):
        assert torch.equal(a, b)
    w["residual"] = m["residual"] = m["residual"].clone().requires_grad_()
    _run_and_compare({**m, "residual": m["residual"].detach()})


def test_empty_calls():
    m = _make(torch.float32, (0, 4, 32))
    names = ("y", "residual", "gate", "post", "pre", "scale")
    leaves = {k: m[k].requires_grad_() for k in names}
    r, x = _call({**m, **leaves})
    assert r.shape == (0, 4, 32) and x.shape == (0, 4, 32)
    grads = torch.autograd.grad((r, x), list(leaves.values()), (m["dr"], m["dx"]))
    assert all((g == 0).all() for g in grads[3:])


def test_graph_and_repeats():
    m = _make(torch.bfloat16, (4, 33, 256))
    want = _call(m)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _call(m)
    for k in ("y", "residual", "gate"):
        m[k].copy_(m[k].flip(0))
    graph.replay()
    assert all(torch.equal(a, b.flip(0)) for a, b in zip(got, want))
    names = ("y", "residual", "gate", "post", "pre", "scale")
    leaves = [m[k].requires_grad_() for k in names]
    runs = [torch.autograd.grad(_call(m), leaves, (m["dr"], m["dx"])) for _ in range(3)]
    assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(r, runs[0]))


def test_refusals():
    from sparseflow_b200.Kernels.block_norm import block_norm
    y, w = torch.zeros(2, 3, 8, device="cuda"), torch.zeros(8, device="cuda")
    for bad in (dict(y=torch.zeros(1, 16385, device="cuda")), dict(post_weight=w[:7]), dict(residual=y[:1]),
                dict(gate=y[..., :1]), dict(gate=y[:1]), dict(gate=y, gate_activation="relu")):
        with pytest.raises(ValueError):
            block_norm(**{"y": y, **bad})
    for bad in (dict(post_weight=w, pre_weight=w.half()), dict(y=y.half(), scale=w.bfloat16()), dict(residual=y.half()),
                dict(gate=y.half()), dict(y=y.double()), dict(residual=y, residual_dtype=torch.float16),
                dict(residual_dtype=torch.bfloat16)):
        with pytest.raises(TypeError):
            block_norm(**{"y": y, **bad})


def test_c_entry_refuses():
    import ctypes
    from sparseflow_b200 import _lib
    lib = _lib.load()
    p = torch.zeros(4096, device="cuda").data_ptr()

    def desc(rows=2, per=1, dim=8, dtype=0, res=0, w=0, gate=0):
        return ctypes.byref(_lib.BlockNormDesc(rows, 8, 8, 8, per, dim, dtype, res, w, gate, 1.0, 1e-6))

    def call(d, y=p, gate=None, out=p):
        return lib.sf_block_norm(y, None, gate, None, None, None, out, None, None, d, None)
    for d in (desc(rows=-1), desc(dim=0), desc(per=0), desc(rows=3, per=2), desc(dtype=4), desc(res=1), desc(w=2),
              desc(gate=4), desc(gate=1)):
        assert call(d) == _lib.SF_ERR_INVALID_ARG
    assert call(desc(), y=None) == _lib.SF_ERR_INVALID_ARG and call(desc(), gate=p) == _lib.SF_ERR_INVALID_ARG
    assert call(desc(), out=None) == _lib.SF_ERR_INVALID_ARG
    assert call(desc(dim=16385)) == _lib.SF_ERR_UNSUPPORTED
    assert lib.sf_block_norm_backward(p, *([None] * 5), p, p, None, p, *([None] * 5), desc(), None, 0, None) == \
        _lib.SF_ERR_WORKSPACE
