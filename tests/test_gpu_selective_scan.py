"""selective_scan and selective_scan_update against the formulas in 64 bits."""
import pytest
import torch

import sequence_reference as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _roundings(length):
    """fp32 roundings of a scan of `length` rows: a step rounds its product and sum, and its decay is off by the
    rounding of the exponent (|dt A| <= 8 here) and a few ulp of dt and of the exponential; a gradient goes through the
    rows twice and multiplies two such values."""
    return 64 * (length + 8)


def _make(dtype, lengths, dim, n, groups, packed, seed=0, gated=True, bias=True, skip=True, state=True, softplus=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = len(lengths)
    lead = (sum(lengths),) if packed else (s, lengths[0])

    def r(*shape, dt=dtype):
        return torch.randn(*shape, device="cuda", generator=g).to(dt)
    f = torch.float32
    off = torch.tensor([0] + torch.tensor(lengths).cumsum(0).tolist(), dtype=torch.int32, device="cuda") if packed else None
    dt = r(*lead, dim) if softplus else r(*lead, dim).abs()
    return dict(x=r(*lead, dim), dt=dt, A=-torch.exp(r(dim, n, dt=f) * 0.5), B=r(*lead, groups, n),
                C=r(*lead, groups, n), D=r(dim, dt=f) if skip else None, z=r(*lead, dim) if gated else None,
                bias=None if not bias else r(dim, dt=f) - 1 if softplus else r(dim, dt=f).abs(), init=r(s, dim, n, dt=f) if state else None, off=off,
                dy=r(*lead, dim), df=r(s, dim, n, dt=f), softplus=softplus)


def _call(m, **kw):
    from sparseflow_b200.Kernels.selective_scan import selective_scan
    return selective_scan(m["x"], m["dt"], m["A"], m["B"], m["C"], m["D"], m["z"], m["bias"], m["softplus"], m["init"],
                          m["off"], True, **kw)


def _run_and_compare(m, final_grad=True):
    names = [k for k in ("x", "dt", "A", "B", "C", "D", "z", "bias", "init") if m[k] is not None]
    leaves = {k: m[k].detach().clone().requires_grad_() for k in names}
    y, f = _call({**m, **leaves})
    with torch.no_grad():
        y2, f2 = _call(m)
    assert torch.equal(y, y2) and torch.equal(f, f2)
    outs, gouts = ((y, f), (m["dy"], m["df"])) if final_grad else ((y,), (m["dy"],))
    grads = dict(zip(names, torch.autograd.grad(outs, list(leaves.values()), gouts)))
    args = (*ref.f64(*(m[k] for k in ("x", "dt", "A", "B", "C", "D", "z", "bias"))), m["softplus"], ref.f64(m["init"]),
            None if m["off"] is None else m["off"].tolist(), ref.f64(m["dy"]), ref.f64(m["df"]) if final_grad else None)
    val, mag = ref.scan(*args), ref.scan(*args, mag=True)
    longest = m["x"].shape[-2] if m["off"] is None else int((m["off"][1:] - m["off"][:-1]).max())
    k = _roundings(longest)
    ref.close(y, val["y"], mag["y"], k, "y")
    ref.close(f, val["final"], mag["final"], k, "final")
    for n in names:
        ref.close(grads[n], val["d" + n], mag["d" + n], 2 * k, n)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, groups, dim", [(1, 1, 7), (3, 2, 30), (4, 1, 64), (8, 1, 33), (13, 2, 70), (16, 1, 96),
                                            (16, 4, 64), (32, 1, 40), (50, 1, 24), (128, 2, 12)])
def test_packed_prompts(dtype, n, groups, dim):
    _run_and_compare(_make(dtype, [5, 0, 1, 37, 16, 0], dim, n, groups, True))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 31, 33, 64, 130])
def test_batched_prompts(dtype, length):
    _run_and_compare(_make(dtype, [length] * 2, 40, 16, 1, False, state=False), final_grad=False)


@pytest.mark.parametrize("part", ["gated", "bias", "skip", "state", "softplus"])
def test_parts_left_out(part):
    _run_and_compare(_make(torch.float32, [20, 20], 48, 16, 1, False, **{part: False}))


def test_long_sequence_and_many_channels():
    """Long enough for any cut along the sequence, states carried over it; compared with 64 bits."""
    _run_and_compare(_make(torch.float32, [1100], 10, 16, 1, False, seed=4))
    _run_and_compare(_make(torch.bfloat16, [700, 3, 600], 520, 4, 1, True, seed=5))


def test_decays_to_nothing_and_not_at_all():
    """dt large enough that exp(dt A) is 0, and 0 so that it is 1."""
    m = _make(torch.float32, [40], 32, 16, 1, False, bias=False, softplus=False)
    m["dt"][0, 10] = 0.0
    m["dt"][0, 20] = 500.0
    m["dt"][0, 21:30] = 0.0
    y, f = _call(m)
    args = ref.f64(*(m[k] for k in ("x", "dt", "A", "B", "C", "D", "z"))) + [None, False, ref.f64(m["init"]), None]
    val, mag = ref.scan(*args), ref.scan(*args, mag=True)
    ref.close(y, val["y"], mag["y"], _roundings(40), "y")
    ref.close(f, val["final"], mag["final"], _roundings(40), "final")


def test_small_steps_keep_their_digits():
    """softplus of a very negative argument, where 1 + e^v loses e^v: dt about 1e-6, over many rows."""
    m = _make(torch.float32, [60], 32, 16, 1, False, state=False, gated=False, skip=False)
    m["dt"] = torch.full_like(m["dt"], -13.8)
    m["bias"] = None
    y, _ = _call(m)
    args = ref.f64(*(m[k] for k in ("x", "dt", "A", "B", "C", "D", "z"))) + [None, True, None, None]
    ref.close(y, ref.scan(*args)["y"], ref.scan(*args, mag=True)["y"], _roundings(60), "y")


@pytest.mark.parametrize("offset, pad", [(0, 8), (8, 24), (3, 2)])
def test_slices_of_wider_rows(offset, pad):
    """x, z, dt, B and C as columns of projections' outputs: the same bits as their copies."""
    m = _make(torch.bfloat16, [45, 45], 64, 16, 1, False)
    w = dict(m)
    for k in ("x", "z", "dt", "B", "C"):
        t = m[k].flatten(2)
        wide = torch.full((2, 45, offset + t.shape[2] + pad), 7.0, device="cuda", dtype=t.dtype)
        wide[..., offset:offset + t.shape[2]] = t
        w[k] = wide[..., offset:offset + t.shape[2]]
        if k in "BC":
            w[k] = w[k].unflatten(2, (1, 16))
    for a, b in zip(_call(w), _call(m)):
        assert torch.equal(a, b)
    w["B"] = m["B"].squeeze(2)  # without the group dimension
    w["x"] = m["x"].transpose(0, 1).contiguous().transpose(0, 1)
    w["z"] = m["z"].transpose(1, 2).contiguous().transpose(1, 2)
    for a, b in zip(_call(w), _call(m)):
        assert torch.equal(a, b)


def test_gradients_by_differences():
    """Along a random direction of each input, from the kernel's own outputs in fp32: differences of step 1e-2 are
    off by their third derivative (1e-4 of the magnitude) and by rounding of the loss (1e-5 / 1e-2)."""
    m = _make(torch.float32, [24, 24], 32, 16, 2, False, seed=9)
    names = ("x", "dt", "A", "B", "C", "D", "z", "bias", "init")

    def loss(m):
        y, f = _call(m)
        return (y.double() * m["dy"]).sum() + (f.double() * m["df"]).sum()
    leaves = {k: m[k].clone().requires_grad_() for k in names}
    grads = torch.autograd.grad(loss({**m, **leaves}), list(leaves.values()))
    g = torch.Generator(device="cuda").manual_seed(1)
    for k, grad in zip(names, grads):
        v = torch.randn(m[k].shape, device="cuda", generator=g)
        v = v / v.norm()
        diff = (loss({**m, k: m[k] + 1e-2 * v}) - loss({**m, k: m[k] - 1e-2 * v})).item() / 2e-2
        want = (grad.double() * v).sum().item()
        assert abs(diff - want) <= 5e-3 * (grad.norm().item() + 1), (k, diff, want)


def test_empty_calls():
    m = _make(torch.float32, [0, 0], 16, 4, 1, False)
    y, f = _call(m)
    assert y.shape == (2, 0, 16) and torch.equal(f, m["init"])
    m = _make(torch.float32, [0, 0], 16, 4, 1, True)
    y, f = _call(m)
    assert y.shape == (0, 16) and torch.equal(f, m["init"])
    m = {**_make(torch.float32, [3], 16, 4, 1, False), "init": None}
    for k in ("x", "dt", "B", "C", "z"):
        m[k] = m[k][:0].clone().requires_grad_()
    m["A"].requires_grad_()
    y, f = _call(m)
    assert y.shape == (0, 3, 16) and f.shape == (0, 16, 4)
    assert (torch.autograd.grad(y, m["A"], torch.zeros_like(y))[0] == 0).all()


def test_wrong_offsets_stay_in_memory():
    m = _make(torch.float32, [10, 20, 5], 32, 16, 1, True)
    good, _ = _call(m)
    m["off"] = torch.tensor([0, 10, 30, 5000], dtype=torch.int32, device="cuda")
    assert torch.equal(_call(m)[0], good)
    m["off"] = torch.tensor([-7, 10, 30, 2], dtype=torch.int32, device="cuda")
    assert torch.equal(_call(m)[0][:30], good[:30])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, groups, dim", [(1, 1, 5), (16, 1, 96), (13, 2, 70), (32, 2, 130), (100, 1, 9)])
def test_single_tokens(dtype, n, groups, dim):
    from sparseflow_b200.Kernels.selective_scan import selective_scan_update
    rows = 11
    m = _make(dtype, [1] * rows, dim, n, groups, False, seed=2)
    pool = torch.randn(rows + 4, dim, n, device="cuda")
    idx = torch.randperm(rows + 4, device="cuda")[:rows].to(torch.int32)
    idx[3], idx[7] = -1, rows + 4
    live = (idx >= 0) & (idx < rows + 4)
    before = pool.clone()
    args = [m["x"][:, 0], m["dt"][:, 0], m["A"], m["B"][:, 0], m["C"][:, 0], pool, m["D"], m["z"][:, 0], m["bias"]]
    y = selective_scan_update(*args, state_indices=idx)
    at = idx[live].long()
    r = ref.f64(*(m[k][live] if k not in ("A", "D", "bias") else m[k] for k in ("x", "dt", "A", "B", "C", "D", "z", "bias")))
    val, mag = (ref.scan(*r, True, ref.f64(before[at]), None, mag=g) for g in (False, True))
    ref.close(y[live], val["y"][:, 0], mag["y"][:, 0], _roundings(1), "y")
    ref.close(pool[at], val["final"], mag["final"], _roundings(1), "state")
    assert (y[~live] == 0).all()
    rest = torch.ones(rows + 4, dtype=torch.bool, device="cuda")
    rest[at] = False
    assert torch.equal(pool[rest], before[rest])
    args[5] = pool = before.clone()
    y = selective_scan_update(*args[:6])  # no indices, no D, no gate, no bias
    r = ref.f64(*(m[k] for k in ("x", "dt", "A", "B", "C")))
    val, mag = (ref.scan(*r, None, None, None, True, ref.f64(before[:rows]), None, mag=g) for g in (False, True))
    ref.close(y, val["y"][:, 0], mag["y"][:, 0], _roundings(1), "y")
    ref.close(pool[:rows], val["final"], mag["final"], _roundings(1), "state")


def test_tokens_continue_a_prompt():
    from sparseflow_b200.Kernels.selective_scan import selective_scan_update
    m = _make(torch.float32, [40, 40], 64, 16, 1, False, state=False)
    y, f = _call(m)
    part = {k: v[:, :32] if k in ("x", "dt", "B", "C", "z") else v for k, v in m.items()}
    y1, state = _call(part)
    outs = [y1]
    for t in range(32, 40):
        row = {k: m[k][:, t] for k in ("x", "dt", "B", "C", "z")}
        outs.append(selective_scan_update(row["x"], row["dt"], m["A"], row["B"], row["C"], state, m["D"], row["z"],
                                          m["bias"])[:, None])
    r = ref.f64(*(m[k] for k in ("x", "dt", "A", "B", "C", "D", "z", "bias")))
    mag = ref.scan(*r, True, None, None, mag=True)
    ref.close(torch.cat(outs, 1), ref.f64(y), mag["y"], 2 * _roundings(40), "y")
    ref.close(state, ref.f64(f), mag["final"], 2 * _roundings(40), "state")


def test_another_stream_and_a_graph():
    m = _make(torch.bfloat16, [64, 64], 128, 16, 1, False)
    want = _call(m)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _call(m)[0]
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _call(m)[0]
    for k in ("x", "dt", "B", "C", "z", "init"):
        m[k].copy_(m[k].flip(0))
    graph.replay()
    assert torch.equal(got, want.flip(0))


def test_gradients_repeat_bit_for_bit():
    m = _make(torch.float32, [300, 300], 200, 16, 1, False)
    names = ("x", "dt", "A", "B", "C", "D", "z", "bias", "init")
    leaves = {k: m[k].requires_grad_() for k in names}
    runs = [torch.autograd.grad(_call({**m, **leaves}), list(leaves.values()), (m["dy"], m["df"])) for _ in range(3)]
    assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(r, runs[0]))


def test_parameters_of_another_type_get_their_gradients():
    m = _make(torch.bfloat16, [20], 32, 16, 1, False)
    A = m["A"].to(torch.bfloat16).requires_grad_()
    y, _ = _call({**m, "A": A})
    assert torch.autograd.grad(y, A, m["dy"])[0].dtype == torch.bfloat16
    assert torch.equal(y, _call({**m, "A": A.detach().float()})[0])


def test_refusals():
    from sparseflow_b200.Kernels.selective_scan import selective_scan, selective_scan_update
    m = _make(torch.float32, [5, 5], 8, 4, 2, False)
    base = {k: m[k] for k in ("x", "dt", "A", "B", "C", "D", "z")}
    z = torch.zeros
    for bad in (dict(A=z(8, 129, device="cuda")), dict(A=z(7, 4, device="cuda")), dict(B=m["B"][:, :4]),
                dict(B=z(2, 5, 3, 4, device="cuda"), C=z(2, 5, 3, 4, device="cuda")), dict(C=m["C"][..., :1, :]),
                dict(dt=m["dt"][..., :1]), dict(D=z(7, device="cuda")), dict(z=m["z"][:1]),
                dict(dt_bias=z(1, device="cuda")), dict(initial_state=z(2, 8, 5, device="cuda")),
                dict(seq_offsets=z(2, dtype=torch.int32, device="cuda")), dict(x=m["x"][0], dt=m["dt"][0])):
        with pytest.raises(ValueError):
            selective_scan(**{**base, **bad})
    for bad in (dict(dt=m["dt"].half()), dict(B=m["B"].half()), dict(z=m["z"].bfloat16()),
                dict(initial_state=z(2, 8, 4, device="cuda").half()), {k: v.double() for k, v in base.items()}):
        with pytest.raises(TypeError):
            selective_scan(**{**base, **bad})
    one = {k: v[:, 0] if k not in "AD" else v for k, v in base.items()}
    with pytest.raises(TypeError):
        selective_scan_update(**one, state=z(2, 8, 4, device="cuda").half())
    with pytest.raises(ValueError):
        selective_scan_update(**one, state=z(1, 8, 4, device="cuda"))
    with pytest.raises(ValueError):
        selective_scan_update(**one, state=z(2, 4, 8, device="cuda").transpose(1, 2))
    with pytest.raises(TypeError):
        selective_scan_update(**one, state=z(2, 8, 4, device="cuda"), state_indices=z(2, device="cuda"))


def test_c_entry_refuses():
    import ctypes
    from sparseflow_b200 import _lib
    lib = _lib.load()
    p = torch.zeros(4096, device="cuda").data_ptr()

    def desc(**kw):
        v = dict(n_seq=1, dim=8, state=4, groups=1, softplus=1, dtype=0, packed=0, **{})
        v.update(kw)
        return ctypes.byref(_lib.SelectiveScanDesc(4, *([0, 8] * 3), *([0, 4] * 2), *v.values()))

    def call(d, x=p, A=p, off=None):
        return lib.sf_selective_scan(x, p, A, p, p, None, None, None, None, off, p, None, None, d, None, 0, None)
    for d in (desc(groups=3), desc(state=0), desc(dtype=5), desc(n_seq=-1), desc(packed=1)):
        assert call(d) == _lib.SF_ERR_INVALID_ARG
    assert call(desc(), x=None) == _lib.SF_ERR_INVALID_ARG and call(desc(), A=None) == _lib.SF_ERR_INVALID_ARG
    assert call(desc(), off=p) == _lib.SF_ERR_INVALID_ARG
    assert call(desc(state=129)) == _lib.SF_ERR_UNSUPPORTED
    assert lib.sf_selective_scan_backward(*([p] * 5), None, None, None, None, p, p, None, p, p, p, p, p, None, None, None,
                                          None, desc(), None, 0, None) == _lib.SF_ERR_WORKSPACE


def test_pool_without_slots_is_all_padding():
    from sparseflow_b200.Kernels.causal_conv1d import causal_conv1d_update
    from sparseflow_b200.Kernels.selective_scan import selective_scan_update
    m = _make(torch.bfloat16, [1] * 3, 24, 16, 1, False)
    idx = torch.tensor([0, -1, 5], dtype=torch.int32, device="cuda")
    y = selective_scan_update(m["x"][:, 0], m["dt"][:, 0], m["A"], m["B"][:, 0], m["C"][:, 0],
                              torch.zeros(0, 24, 16, device="cuda"), m["D"], state_indices=idx)
    assert y.shape == (3, 24) and (y == 0).all()
    x = m["x"][:, 0].contiguous()
    y = causal_conv1d_update(x, x.new_zeros(0, 3, 24), x.new_ones(24, 4), state_indices=idx)
    assert y.shape == (3, 24) and (y == 0).all()
