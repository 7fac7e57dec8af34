"""causal_conv1d and causal_conv1d_update against the formulas in 64 bits."""
import pytest
import torch

import sequence_reference as ref

pytestmark = pytest.mark.gpu

# fp32 roundings an output passes through: width products and additions, the bias, the activation (its exponential
# and division are good to a few ulp); a gradient goes through them twice and is summed over at most so many rows.
FWD = 8 + 12
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _make(dtype, lengths, dim, width, packed, seed=0, wdtype=None, bias=True, state=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = len(lengths)
    shape = (sum(lengths), dim) if packed else (n, lengths[0], dim)

    def r(*s, dt=dtype):
        return torch.randn(*s, device="cuda", generator=g).to(dt)
    wdtype = wdtype or dtype
    off = torch.tensor([0] + torch.tensor(lengths).cumsum(0).tolist(), dtype=torch.int32, device="cuda") if packed else None
    return dict(x=r(*shape), weight=r(dim, width, dt=wdtype), bias=r(dim, dt=wdtype) if bias else None,
                init=r(n, width - 1, dim) if state else None, off=off, dy=r(*shape), df=r(n, width - 1, dim))


def _run_and_compare(m, act, roundings):
    from sparseflow_b200.Kernels.causal_conv1d import causal_conv1d
    leaves = {k: m[k].detach().requires_grad_() for k in ("x", "weight", "bias", "init") if m[k] is not None}
    y, f = causal_conv1d(leaves["x"], leaves["weight"], leaves.get("bias"), act, leaves.get("init"), m["off"], True)
    with torch.no_grad():  # the same call without gradients gives the same bits
        y2, f2 = causal_conv1d(m["x"], m["weight"], m["bias"], act, m["init"], m["off"], True)
    assert torch.equal(y, y2) and torch.equal(f, f2)
    grads = dict(zip(leaves, torch.autograd.grad((y, f), list(leaves.values()), (m["dy"], m["df"]))))
    args = (*ref.f64(m["x"], m["weight"], m["bias"]), act == "silu", ref.f64(m["init"]),
            None if m["off"] is None else m["off"].tolist(), *ref.f64(m["dy"], m["df"]))
    val, mag = ref.conv(*args), ref.conv(*args, mag=True)
    ref.close(y, val[0], mag[0], FWD, "y")
    assert torch.equal(f.double().cpu(), val[1])  # rows are copied
    for i, k in ((2, "x"), (3, "weight"), (4, "bias"), (5, "init")):
        if k in grads:
            ref.close(grads[k], val[i], mag[i], roundings, k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [2, 3, 4, 5, 8])
@pytest.mark.parametrize("act", [None, "silu"])
@pytest.mark.parametrize("dim", [1, 24, 77, 1032])
def test_packed_prompts(dtype, width, act, dim):
    lengths = [3, 0, 1, 70, 33, 0]
    _run_and_compare(_make(dtype, lengths, dim, width, True), act, 2 * FWD + sum(lengths))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("length", [1, 2, 31, 32, 33, 64, 65, 200])
@pytest.mark.parametrize("state", [False, True])
def test_batched_prompts(dtype, length, state):
    _run_and_compare(_make(dtype, [length] * 3, 136, 4, False, state=state), "silu", 2 * FWD + 3 * length)


def test_parameters_in_32_bits_and_no_bias():
    _run_and_compare(_make(torch.bfloat16, [40, 9], 64, 4, True, wdtype=torch.float32, bias=False), "silu", 2 * FWD + 49)


def test_wide_and_many():
    """More slots than blocks side by side, several blocks of channels."""
    _run_and_compare(_make(torch.bfloat16, [700, 1300], 2056, 4, True), "silu", 2 * FWD + 2000)


@pytest.mark.parametrize("offset, pad", [(0, 8), (8, 16), (3, 5)])
def test_slices_of_wider_rows(offset, pad):
    """x as columns of a projection's output: the same bits as its copy, gradients into the slice."""
    from sparseflow_b200.Kernels.causal_conv1d import causal_conv1d
    m = _make(torch.bfloat16, [50, 50], 64, 4, False)
    wide = torch.zeros(2, 50, offset + 64 + pad, device="cuda", dtype=torch.bfloat16)
    wide[..., offset:offset + 64] = m["x"]
    x = wide[..., offset:offset + 64]
    assert torch.equal(causal_conv1d(x, m["weight"], m["bias"], "silu"),
                       causal_conv1d(m["x"], m["weight"], m["bias"], "silu"))
    turned = m["x"].transpose(1, 2).contiguous().transpose(1, 2)  # channels not contiguous
    assert torch.equal(causal_conv1d(turned, m["weight"], m["bias"]), causal_conv1d(m["x"], m["weight"], m["bias"]))
    both = torch.randn(50, 2, 64, device="cuda").to(torch.bfloat16).transpose(0, 1)  # rows of two sequences in turn
    assert torch.equal(causal_conv1d(both, m["weight"]), causal_conv1d(both.contiguous(), m["weight"]))


def test_infinities_stay_where_the_taps_reach():
    from sparseflow_b200.Kernels.causal_conv1d import causal_conv1d
    x = torch.zeros(1, 40, 8, device="cuda")
    x[0, 10, 3] = float("inf")
    x[0, 20, 4] = float("nan")
    y = causal_conv1d(x, torch.ones(8, 3, device="cuda"))
    assert torch.isinf(y[0, 10:13, 3]).all() and torch.isnan(y[0, 20:23, 4]).all()
    y[0, 10:13, 3] = 0
    y[0, 20:23, 4] = 0
    assert (y == 0).all()


def test_empty_calls():
    from sparseflow_b200.Kernels.causal_conv1d import causal_conv1d, causal_conv1d_update
    w = torch.randn(8, 4, device="cuda", requires_grad=True)
    for shape in ((0, 5, 8), (2, 0, 8)):
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        y = causal_conv1d(x, w)
        assert y.shape == x.shape
        gx, gw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
        assert gx.shape == x.shape and (gw == 0).all()
    init = torch.randn(2, 3, 8, device="cuda")
    y, f = causal_conv1d(torch.zeros(2, 0, 8, device="cuda"), w.detach(), initial_state=init, return_final_state=True)
    assert torch.equal(f, init)
    y, f = causal_conv1d(torch.zeros(0, 8, device="cuda"), w.detach(), return_final_state=True,
                         seq_offsets=torch.zeros(3, dtype=torch.int32, device="cuda"))
    assert y.shape == (0, 8) and (f == 0).all() and f.shape == (2, 3, 8)
    assert causal_conv1d_update(torch.zeros(0, 8, device="cuda"), init, w.detach()).shape == (0, 8)


def test_wrong_offsets_stay_in_memory():
    """Offsets past the rows, or falling ones, are clamped: every other sequence is still right."""
    from sparseflow_b200.Kernels.causal_conv1d import causal_conv1d
    m = _make(torch.float32, [10, 20, 5], 64, 4, True, state=False)
    good = causal_conv1d(m["x"], m["weight"], seq_offsets=m["off"])
    off = torch.tensor([0, 10, 30, 5000], dtype=torch.int32, device="cuda")
    assert torch.equal(causal_conv1d(m["x"], m["weight"], seq_offsets=off), good)
    off = torch.tensor([-7, 10, 30, 2], dtype=torch.int32, device="cuda")
    assert torch.equal(causal_conv1d(m["x"], m["weight"], seq_offsets=off)[:30], good[:30])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [2, 4, 7])
@pytest.mark.parametrize("rows, dim", [(1, 5), (3, 64), (67, 1032)])
def test_single_tokens(dtype, width, rows, dim):
    from sparseflow_b200.Kernels.causal_conv1d import causal_conv1d_update
    g = torch.Generator(device="cuda").manual_seed(3)
    pool = torch.randn(rows + 5, width - 1, dim, device="cuda", generator=g).to(dtype)
    x = torch.randn(rows, dim, device="cuda", generator=g).to(dtype)
    w = torch.randn(dim, width, device="cuda", generator=g).to(dtype)
    b = torch.randn(dim, device="cuda", generator=g).to(dtype)
    idx = torch.randperm(rows + 5, device="cuda", generator=g)[:rows].to(torch.int32)
    idx[rows // 2] = -1
    live = idx >= 0
    before = pool.clone()
    y = causal_conv1d_update(x, pool, w, b, "silu", idx)
    assert (y[~live] == 0).all()
    at = idx[live].long()
    args = (*ref.f64(x[live][:, None], w, b), True, ref.f64(before[at]), None)
    val, mag = ref.conv(*args), ref.conv(*args, mag=True)
    ref.close(y[live], val[0][:, 0], mag[0][:, 0], FWD, "y")
    want = before.clone()
    want[at] = torch.cat([before[at][:, 1:], x[live][:, None]], 1)
    assert torch.equal(pool, want)
    # an index past the pool is padding too, and no indices mean slot i for row i
    idx2 = torch.full_like(idx, rows + 5)
    assert (causal_conv1d_update(x, pool, w, b, "silu", idx2) == 0).all() and torch.equal(pool, want)
    first = pool[:rows].clone()
    y0 = causal_conv1d_update(x, pool, w, b)
    assert torch.equal(pool[:rows], torch.cat([first[:, 1:], x[:, None]], 1)) and torch.isfinite(y0.float()).all()


def test_tokens_continue_a_prompt():
    from sparseflow_b200.Kernels.causal_conv1d import causal_conv1d, causal_conv1d_update
    m = _make(torch.bfloat16, [37, 37], 72, 4, False, state=False)
    whole = causal_conv1d(m["x"], m["weight"], m["bias"], "silu")
    y, state = causal_conv1d(m["x"][:, :30], m["weight"], m["bias"], "silu", return_final_state=True)
    assert torch.equal(y, whole[:, :30])
    for t in range(30, 37):
        assert torch.equal(causal_conv1d_update(m["x"][:, t], state, m["weight"], m["bias"], "silu"), whole[:, t])


def test_another_stream_and_a_graph():
    from sparseflow_b200.Kernels.causal_conv1d import causal_conv1d
    m = _make(torch.bfloat16, [64, 64], 256, 4, False)
    want = causal_conv1d(m["x"], m["weight"], m["bias"], "silu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = causal_conv1d(m["x"], m["weight"], m["bias"], "silu")
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = causal_conv1d(m["x"], m["weight"], m["bias"], "silu")
    m["x"].copy_(m["x"].flip(0))
    graph.replay()
    assert torch.equal(got, want.flip(0))


def test_gradients_repeat_bit_for_bit():
    from sparseflow_b200.Kernels.causal_conv1d import causal_conv1d
    m = _make(torch.float32, [513, 513], 200, 4, False, state=False)
    leaves = [m[k].requires_grad_() for k in ("x", "weight", "bias")]
    runs = [torch.autograd.grad(causal_conv1d(*leaves, "silu"), leaves, m["dy"]) for _ in range(3)]
    assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(r, runs[0]))


def test_refusals():
    from sparseflow_b200.Kernels.causal_conv1d import causal_conv1d, causal_conv1d_update
    x, w = torch.zeros(2, 5, 8, device="cuda"), torch.zeros(8, 4, device="cuda")
    off = torch.tensor([0, 5], dtype=torch.int32, device="cuda")
    for bad in (dict(weight=torch.zeros(8, 1, device="cuda")), dict(weight=torch.zeros(8, 9, device="cuda")),
                dict(weight=torch.zeros(7, 4, device="cuda")), dict(bias=torch.zeros(7, device="cuda")),
                dict(activation="tanh"), dict(initial_state=torch.zeros(2, 4, 8, device="cuda")),
                dict(seq_offsets=off), dict(x=x[0]), dict(x=x[0], seq_offsets=off[None])):
        with pytest.raises(ValueError):
            causal_conv1d(**{"x": x, "weight": w, **bad})
    for bad in (dict(bias=torch.zeros(8, device="cuda").half()), dict(x=x.double()), dict(x=x[0], seq_offsets=off.long()),
                dict(initial_state=torch.zeros(2, 3, 8, device="cuda").half())):
        with pytest.raises(TypeError):
            causal_conv1d(**{"x": x, "weight": w, **bad})
    state = torch.zeros(3, 3, 8, device="cuda")
    with pytest.raises(ValueError):
        causal_conv1d_update(x, state, w)
    with pytest.raises(ValueError):
        causal_conv1d_update(x[:, 0], state[:1], w)
    with pytest.raises(ValueError):
        causal_conv1d_update(x[:, 0], state.transpose(1, 2).contiguous().transpose(1, 2), w)
    with pytest.raises(TypeError):
        causal_conv1d_update(x[:, 0], state, w, state_indices=torch.zeros(2, dtype=torch.int64, device="cuda"))


def test_c_entry_refuses():
    """Status codes of the C entry, nothing launched."""
    import ctypes
    from sparseflow_b200 import _lib
    lib = _lib.load()
    x = torch.zeros(1, 4, 8, device="cuda")
    w = torch.zeros(8, 4, device="cuda")

    def call(x=x.data_ptr(), w=w.data_ptr(), off=None, y=x.data_ptr(), **kw):
        d = _lib.CausalConv1dDesc(4, 32, 8, 1, 8, kw.get("width", 4), 0, kw.get("dtype", 0), 0, kw.get("packed", 0))
        return lib.sf_causal_conv1d(x, w, None, None, off, y, None, ctypes.byref(d), None)
    assert call(w=None) == _lib.SF_ERR_INVALID_ARG
    assert call(x=None) == _lib.SF_ERR_INVALID_ARG
    assert call(width=9) == _lib.SF_ERR_INVALID_ARG and call(width=1) == _lib.SF_ERR_INVALID_ARG
    assert call(dtype=7) == _lib.SF_ERR_INVALID_ARG and call(packed=1) == _lib.SF_ERR_INVALID_ARG
    d = _lib.CausalConv1dDesc(4, 32, 8, 1, 8, 4, 0, 0, 0, 0)
    p = x.data_ptr()
    assert lib.sf_causal_conv1d_backward(p, w.data_ptr(), None, None, None, p, None, p, w.data_ptr(), None, None,
                                         ctypes.byref(d), None, 0, None) == _lib.SF_ERR_WORKSPACE
