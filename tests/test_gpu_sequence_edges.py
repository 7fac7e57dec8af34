"""The sequence operators where a call is most easily wrong: many taps, memory beside the outputs, empty and unaligned
tensors, batches past a grid's limits."""
import ctypes

import pytest
import torch

import sequence_reference as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
CONV_FWD = 8 + 12  # fp32 roundings of a convolution's output: taps, bias and activation


def _offsets(lengths):
    return torch.tensor([0] + torch.tensor(lengths).cumsum(0).tolist(), dtype=torch.int32, device="cuda")


# ----------------------------------------------------------------------------------------------------------------------
# causal_conv1d
# ----------------------------------------------------------------------------------------------------------------------

def _conv_gradients(dtype, lengths, dim, width, packed):
    """Every output and gradient of a convolution with a SiLU, initial and final state, against 64 bits."""
    from sparseflow_b200.Kernels.causal_conv1d import causal_conv1d
    g = torch.Generator(device="cuda").manual_seed(width)

    def r(*s):
        return torch.randn(*s, device="cuda", generator=g).to(dtype)
    n = len(lengths)
    shape = (sum(lengths), dim) if packed else (n, lengths[0], dim)
    off = _offsets(lengths) if packed else None
    x, w, b, init, dy, df = r(*shape), r(dim, width), r(dim), r(n, width - 1, dim), r(*shape), r(n, width - 1, dim)
    leaves = [t.requires_grad_() for t in (x, w, b, init)]
    outs = causal_conv1d(x, w, b, "silu", init, off, True)
    grads = torch.autograd.grad(outs, leaves, (dy, df))
    args = (*ref.f64(x, w, b), True, ref.f64(init), None if off is None else off.tolist(), *ref.f64(dy, df))
    val, mag = ref.conv(*args), ref.conv(*args, mag=True)
    ref.close(outs[0], val[0], mag[0], CONV_FWD, "y")
    for i, (name, got) in enumerate(zip(("dx", "dweight", "dbias", "dinit"), grads)):
        ref.close(got, val[2 + i], mag[2 + i], 2 * CONV_FWD + sum(lengths), name)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [5, 6, 7, 8])
def test_many_taps_over_many_slots(dtype, width):
    """More slots, and sequences that begin inside the packed rows, than run on the GPU at a time: a gradient's row is
    stored by its own slot alone."""
    _conv_gradients(dtype, [9 + 7 * i % 13 for i in range(5000)], 16, width, True)
    _conv_gradients(dtype, [21] * 2500, 9, width, False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [5, 6, 7, 8])
@pytest.mark.parametrize("length", [8, 12, 130, 1029])
def test_many_taps_long_sequences(dtype, width, length):
    _conv_gradients(dtype, [length] * 2, 136, width, False)
    _conv_gradients(dtype, [length, 1, length + 3], 136, width, True)


@pytest.mark.parametrize("width", range(2, 9))
@pytest.mark.parametrize("length", [1, 4, 8, 131])
def test_conv_writes_its_outputs_alone(width, length):
    """Outputs in the middle of larger buffers given to the C entries: what lies before and after stays."""
    from sparseflow_b200 import _lib
    lib, dim, n, pad = _lib.load(), 24, 3, 8 * 24
    sizes = {"y": n * length * dim, "final": n * (width - 1) * dim, "dx": n * length * dim, "dw": dim * width, "db": dim,
             "dinit": n * (width - 1) * dim}
    buffers = {k: torch.full((pad + s + pad,), -77.0, device="cuda") for k, s in sizes.items()}
    at = {k: b.data_ptr() + 4 * pad for k, b in buffers.items()}
    x, dy = (torch.randn(n, length, dim, device="cuda") for _ in range(2))
    w, b = torch.randn(dim, width, device="cuda"), torch.randn(dim, device="cuda")
    init, df = (torch.randn(n, width - 1, dim, device="cuda") for _ in range(2))
    d = ctypes.byref(_lib.CausalConv1dDesc(length, length * dim, dim, n, dim, width, 1, 0, 0, 0))
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.sf_causal_conv1d(x.data_ptr(), w.data_ptr(), b.data_ptr(), init.data_ptr(), None, at["y"], at["final"], d,
                                stream) == _lib.SF_OK
    nbytes = lib.sf_causal_conv1d_backward_workspace_size(d)
    ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    assert lib.sf_causal_conv1d_backward(x.data_ptr(), w.data_ptr(), b.data_ptr(), init.data_ptr(), None, dy.data_ptr(),
                                         df.data_ptr(), at["dx"], at["dw"], at["db"], at["dinit"], d, ws.data_ptr(),
                                         nbytes, stream) == _lib.SF_OK
    for k, buf in buffers.items():
        assert (buf[:pad] == -77).all() and (buf[-pad:] == -77).all(), k
    val = ref.conv(*ref.f64(x, w, b), True, ref.f64(init), None, *ref.f64(dy, df))
    mag = ref.conv(*ref.f64(x, w, b), True, ref.f64(init), None, *ref.f64(dy, df), mag=True)
    dx = buffers["dx"][pad:-pad].view(n, length, dim)
    ref.close(dx, val[2], mag[2], 2 * CONV_FWD + n * length, "dx")


# ----------------------------------------------------------------------------------------------------------------------
# block_norm
# ----------------------------------------------------------------------------------------------------------------------

def _norm_leaves(shape, gate_shape):
    def r(*s):
        return torch.randn(*s, device="cuda").requires_grad_()
    dim = shape[-1]
    return dict(y=r(*shape), residual=r(*shape), gate=r(*gate_shape), post_weight=r(dim), pre_weight=r(dim), scale=r(dim))


def test_norm_of_no_sequences_with_a_gate_each():
    """No sequences of five rows: no gate rows either, and the weights' gradients are 0."""
    from sparseflow_b200.Kernels.block_norm import block_norm
    leaves = _norm_leaves((0, 5, 32), (0, 1, 32))
    r, x = block_norm(**leaves, gate_activation="silu")
    grads = torch.autograd.grad((r, x), list(leaves.values()), (torch.ones_like(r), torch.ones_like(x)))
    assert all(g.shape == t.shape and (g == 0).all() for g, t in zip(grads, leaves.values()))


def test_norm_gates_of_empty_sequences():
    """Sequences without rows: their gates' gradient is 0, whatever the memory held before."""
    from sparseflow_b200.Kernels.block_norm import block_norm
    leaves = _norm_leaves((3, 0, 64), (3, 1, 64))
    r, x = block_norm(**leaves, gate_activation="sigmoid")
    used = [torch.full((3, 1, 64), float("nan"), device="cuda") for _ in range(8)]
    del used  # the allocator gives such a block next
    grads = torch.autograd.grad((r, x), list(leaves.values()), (torch.ones_like(r), torch.ones_like(x)))
    assert all(g.shape == t.shape and (g == 0).all() for g, t in zip(grads, leaves.values()))


@pytest.mark.parametrize("dim", [16, 9])
def test_norm_gates_of_many_sequences(dim):
    """More gates than a grid has blocks in its second dimension, forward and backward."""
    from sparseflow_b200.Kernels.block_norm import block_norm
    torch.manual_seed(1)
    leaves = _norm_leaves((70000, 2, dim), (70000, 1, dim))
    dr, dx = torch.randn(70000, 2, dim, device="cuda"), torch.randn(70000, 2, dim, device="cuda")
    r, x = block_norm(**leaves, gate_activation="silu", eps=1e-5)
    grads = torch.autograd.grad((r, x), list(leaves.values()), (dr, dx))
    args = (*ref.f64(*(leaves[k] for k in ("y", "residual", "gate"))), "silu",
            *ref.f64(*(leaves[k] for k in ("post_weight", "pre_weight", "scale"))), 1.0, 1e-5, *ref.f64(dr, dx))
    val, mag = ref.norm(*args), ref.norm(*args, mag=True)
    ref.close(x, val["x"], mag["x"], 64, "normed")
    for name, got, k in zip(leaves, grads, ("dy", "dres", "dgate", "dpost", "dpre", "dscale")):
        ref.close(got, val[k], mag[k], 4 * 64 + (140000 if k in ("dpost", "dpre", "dscale") else 2), name)


# ----------------------------------------------------------------------------------------------------------------------
# selective_scan
# ----------------------------------------------------------------------------------------------------------------------

def _shifted(t, by=1):
    """The same values, contiguous, `by` elements into a buffer: not at a multiple of 16 bytes."""
    buf = torch.empty(t.numel() + 4, dtype=t.dtype, device=t.device)
    out = buf[by:by + t.numel()].view(t.shape)
    out.copy_(t)
    assert out.is_contiguous() and out.data_ptr() % 16
    return out


def _scan_inputs(lead, dim, n, groups=1, dtype=torch.float32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def r(*s, dt=dtype):
        return torch.randn(*s, device="cuda", generator=g).to(dt)
    f = torch.float32
    return dict(x=r(*lead, dim), dt=r(*lead, dim), A=-torch.exp(0.5 * r(dim, n, dt=f)), B=r(*lead, groups, n),
                C=r(*lead, groups, n), D=r(dim, dt=f), z=r(*lead, dim), dt_bias=r(dim, dt=f) - 1)


@pytest.mark.parametrize("n", [3, 4, 13, 16, 64])
@pytest.mark.parametrize("length", [7, 700])
def test_scan_of_unaligned_states(n, length):
    """A, initial states and the gradient of the final states that begin between words of 16 bytes: the same bits."""
    from sparseflow_b200.Kernels.selective_scan import selective_scan
    m = _scan_inputs((2, length), 22, n)
    init, df = torch.randn(2, 22, n, device="cuda"), torch.randn(2, 22, n, device="cuda")
    dy = torch.randn_like(m["x"])

    def run(A, init, df):
        leaves = [A.detach().requires_grad_(), init.detach().requires_grad_(), m["x"].detach().requires_grad_()]
        y, f = selective_scan(**{**m, "A": leaves[0], "x": leaves[2]}, initial_state=leaves[1], return_final_state=True)
        return y, f, *torch.autograd.grad((y, f), leaves, (dy, df))
    want = run(m["A"], init, df)
    for k in range(8):
        got = run(_shifted(m["A"]) if k & 1 else m["A"], _shifted(init, 3) if k & 2 else init,
                  _shifted(df, 2) if k & 4 else df)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), k


@pytest.mark.parametrize("n", [13, 16])
def test_scan_of_a_layer_of_stacked_states(n):
    """Layers of one pool and of stacked parameters, and final states that are joined: ordinary views."""
    from sparseflow_b200.Kernels.selective_scan import selective_scan, selective_scan_update
    m = _scan_inputs((3, 9), 770, n, groups=2)
    stack = torch.stack([m["A"], 2 * m["A"], m["A"]])
    states = torch.randn(4, 3, 770, n, device="cuda")
    one = {k: v if k in ("A", "D", "dt_bias") else v[:, 0] for k, v in m.items()}
    for layer in range(3):
        want_state = states[layer + 1].clone()
        want = selective_scan_update(**{**one, "A": stack[layer].clone()}, state=want_state)
        before = states.clone()
        got = selective_scan_update(**{**one, "A": stack[layer]}, state=states[layer + 1])
        assert torch.equal(got, want) and torch.equal(states[layer + 1], want_state)
        rest = [i for i in range(4) if i != layer + 1]
        assert torch.equal(states[rest], before[rest])
    x = m["x"].requires_grad_()
    finals = [selective_scan(**m, initial_state=s, return_final_state=True)[1] for s in states[1:3]]
    assert torch.autograd.grad(torch.cat([finals[0][:1], finals[1]]).square().sum(), x)[0].isfinite().all()


@pytest.mark.parametrize("n", [3, 13, 16])
def test_tokens_of_unaligned_pools(n):
    from sparseflow_b200.Kernels.selective_scan import selective_scan_update
    m = {k: v if k in ("A", "D", "dt_bias") else v[:, 0] for k, v in _scan_inputs((5, 1), 38, n).items()}
    pool = torch.randn(7, 38, n, device="cuda")
    idx = torch.tensor([6, 0, -1, 3, 2], dtype=torch.int32, device="cuda")
    there = _shifted(pool)
    want = selective_scan_update(**m, state=pool, state_indices=idx)
    assert torch.equal(selective_scan_update(**m, state=there, state_indices=idx), want) and torch.equal(there, pool)
    assert torch.equal(selective_scan_update(**{**m, "A": _shifted(m["A"], 3)}, state=there.clone(), state_indices=idx),
                       selective_scan_update(**m, state=pool, state_indices=idx))


def test_many_rows_of_tokens():
    """More rows than a grid has blocks in its second dimension; past the limit a clear refusal."""
    from sparseflow_b200._lib import SparseFlowError
    from sparseflow_b200.Kernels.selective_scan import selective_scan, selective_scan_update
    m = {k: v if k in ("A", "D", "dt_bias") else v[:, 0] for k, v in _scan_inputs((70001, 1), 5, 3).items()}
    pool = torch.randn(70001, 5, 3, device="cuda")
    parts = pool.clone()
    y = selective_scan_update(**m, state=pool)
    for a, b in ((0, 40000), (40000, 70001)):
        rows = {k: v if k in ("A", "D", "dt_bias") else v[a:b] for k, v in m.items()}
        assert torch.equal(selective_scan_update(**rows, state=parts[a:b]), y[a:b])
    assert torch.equal(pool, parts)
    m = {k: v if k in ("A", "D", "dt_bias") else v[:1].expand(262141, *v.shape[1:]) for k, v in m.items()}
    with pytest.raises(SparseFlowError):
        selective_scan_update(**m, state=torch.zeros(262141, 5, 3, device="cuda"))
    m = _scan_inputs((65536, 1), 2, 1)
    with pytest.raises(SparseFlowError):
        selective_scan(**m)


def _scan_against_64_bits(m, softplus, init, dy, df, length):
    """Outputs and gradients; 64 roundings a row and twice that for gradients (|dt A| <= 8)."""
    from sparseflow_b200.Kernels.selective_scan import selective_scan
    names = ("x", "dt", "A", "B", "C", "D", "z", "dt_bias")
    leaves = {k: m[k].detach().requires_grad_() for k in names if m[k] is not None}
    init = init.requires_grad_()
    outs = selective_scan(**{**m, **leaves}, dt_softplus=softplus, initial_state=init, return_final_state=True)
    grads = torch.autograd.grad(outs, [*leaves.values(), init], (dy, df))
    args = (*ref.f64(*(m[k] for k in names)), softplus, ref.f64(init), None, *ref.f64(dy, df))
    val, mag = ref.scan(*args), ref.scan(*args, mag=True)
    k = 64 * (length + 8)
    ref.close(outs[0], val["y"], mag["y"], k, "y")
    ref.close(outs[1], val["final"], mag["final"], k, "final")
    for name, got in zip([*leaves, "init"], grads):
        name = "bias" if name == "dt_bias" else name
        ref.close(got, val["d" + name], mag["d" + name], 2 * k, name)


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("length", [20, 51, 1100])
def test_scan_of_states_that_grow(sign, length):
    """exp(dt A) = exp(7) a row, by A or by dt: a tile's or a segment's product is past fp32, but the states before the
    first x and the gradients after the last dy are 0, and stay it."""
    m = _scan_inputs((2, length), 10, 16)
    m.update(A=torch.full((10, 16), float(sign), device="cuda"), dt=torch.full_like(m["x"], 7.0 * sign), dt_bias=None)
    m["x"][:, :-3] = 0
    dy = torch.randn_like(m["x"])
    dy[:, 3:] = 0
    _scan_against_64_bits(m, False, torch.zeros(2, 10, 16, device="cuda"), dy, torch.zeros(2, 10, 16, device="cuda"),
                          length)


def test_scan_of_a_small_state_that_grows():
    """16 rows of exp(7) each: the product of a tile is past fp32, a state of 1e-30 after it is not."""
    from sparseflow_b200.Kernels.selective_scan import selective_scan
    m = _scan_inputs((2, 16), 10, 16)
    m.update(A=torch.ones(10, 16, device="cuda"), dt=torch.full_like(m["x"], 7.0), x=torch.zeros_like(m["x"]), dt_bias=None)
    init = 1e-30 * torch.randn(2, 10, 16, device="cuda")
    y, f = selective_scan(**m, dt_softplus=False, initial_state=init, return_final_state=True)
    args = (*ref.f64(*(m[k] for k in ("x", "dt", "A", "B", "C", "D", "z"))), None, False, ref.f64(init), None)
    val, mag = ref.scan(*args), ref.scan(*args, mag=True)
    ref.close(y, val["y"], mag["y"], 64 * 24, "y")
    ref.close(f, val["final"], mag["final"], 64 * 24, "final")


# ----------------------------------------------------------------------------------------------------------------------
# All of them
# ----------------------------------------------------------------------------------------------------------------------

def test_empty_views_of_other_orders():
    """An empty chunk of channels-first activations is an empty call, with gradients."""
    from sparseflow_b200.Kernels.causal_conv1d import causal_conv1d
    from sparseflow_b200.Kernels.selective_scan import selective_scan
    x = torch.randn(2, 8, 5, device="cuda", requires_grad=True)
    bc = torch.randn(2, 4, 5, device="cuda", requires_grad=True)
    part, part_bc = x.transpose(1, 2)[:, :0], bc.transpose(1, 2)[:, :0]
    w = torch.randn(8, 4, device="cuda", requires_grad=True)
    A = -torch.rand(8, 4, device="cuda")
    y, f = causal_conv1d(part, w, return_final_state=True)
    assert y.shape == (2, 0, 8) and (f == 0).all()
    assert (torch.autograd.grad((y, f), (x, w), (y, f), allow_unused=True)[1] == 0).all()
    y, f = selective_scan(part, part, A, part_bc, part_bc, z=part, return_final_state=True)
    assert y.shape == (2, 0, 8) and (f == 0).all()
    assert all((g == 0).all() for g in torch.autograd.grad((y, f), (x, bc), (y, f)))


def test_pools_count_as_written():
    """A state that a backward pass has saved and a token has moved since: autograd's error, not a wrong gradient."""
    from sparseflow_b200.Kernels.causal_conv1d import causal_conv1d, causal_conv1d_update
    from sparseflow_b200.Kernels.selective_scan import selective_scan_update
    x, w = torch.randn(2, 5, 8, device="cuda"), torch.randn(8, 4, device="cuda", requires_grad=True)
    state = torch.randn(2, 3, 8, device="cuda")
    y = causal_conv1d(x, w, initial_state=state)
    with torch.no_grad():
        causal_conv1d_update(x[:, 0], state, w)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    pool, A, b = torch.randn(2, 8, 4, device="cuda"), -torch.rand(8, 4, device="cuda"), torch.randn(2, 4, device="cuda")
    before = pool._version
    selective_scan_update(x[:, 0], x[:, 0], A, b, b, pool)
    assert pool._version > before
    with torch.inference_mode():
        selective_scan_update(x[:, 0], x[:, 0], A, b, b, pool.clone())


def test_backward_through_tokens_raises():
    """Tokens have no gradient: their results say so where a backward pass comes to them, and are the same."""
    from sparseflow_b200.Kernels.causal_conv1d import causal_conv1d_update
    from sparseflow_b200.Kernels.selective_scan import selective_scan_update
    from sparseflow_b200.Ops.state_space import StateSpaceMixer
    x, w, state = torch.randn(2, 8, device="cuda"), torch.randn(8, 4, device="cuda"), torch.randn(2, 3, 8, device="cuda")
    want, moved = causal_conv1d_update(x, before := state.clone(), w), before
    y = causal_conv1d_update(x, state, w.requires_grad_())
    assert torch.equal(y, want) and torch.equal(state, moved)
    with pytest.raises(RuntimeError, match="causal_conv1d_update has no gradient"):
        y.sum().backward()
    A, b = -torch.rand(8, 4, device="cuda"), torch.randn(2, 4, device="cuda")
    pool, same = torch.zeros(2, 8, 4, device="cuda"), torch.zeros(2, 8, 4, device="cuda")
    want = selective_scan_update(x, x, A, b, b, same)
    y = selective_scan_update(x.requires_grad_(), x, A, b, b, pool)
    assert torch.equal(y, want) and torch.equal(pool, same)
    with pytest.raises(RuntimeError, match="selective_scan_update has no gradient"):
        (y * 2).sum().backward()
    with torch.no_grad():
        assert not selective_scan_update(x, x, A, b, b, pool).requires_grad
    m = StateSpaceMixer(16).cuda()
    with pytest.raises(RuntimeError, match="has no gradient"):
        m.step(torch.randn(2, 16, device="cuda"), m.new_state(2)).sum().backward()


def test_model_in_16_bits():
    """A model cast as a whole trains and serves, and its steps equal its prompt."""
    from sparseflow_b200.snn import SpikingStateSpaceLM
    torch.manual_seed(0)
    m = SpikingStateSpaceLM(vocab=40, dim=64, layers=2).cuda().bfloat16()
    tokens = torch.randint(0, 40, (3, 20), device="cuda")
    torch.nn.functional.cross_entropy(m(tokens[:, :-1]).flatten(0, 1).float(), tokens[:, 1:].flatten()).backward()
    assert all(p.grad.dtype == p.dtype and torch.isfinite(p.grad).all() for p in m.parameters())
    assert m.mixers[0].dt_bias.grad.dtype == torch.float32
    with torch.no_grad():
        whole = m(tokens).float()
        logits, states = m.prefill(tokens[:, :12])
        parts = [logits] + [m.step(tokens[:, t], states)[:, None] for t in range(12, 20)]
    # Matrix products of one row and of many may round bf16 values to the one or the other neighbour.
    assert (torch.cat(parts, 1).float() - whole).norm() <= 0.03 * whole.norm()


# ----------------------------------------------------------------------------------------------------------------------
# Bounds that follow the errors, and memory beside outputs
# ----------------------------------------------------------------------------------------------------------------------

ULP = 2.0 ** -24


def _scan_with_bounds(x, dt, A, B, C, D, z):
    """y and the final states in 64 bits [length, dim(, state)], and what fp32 can be off by, row after row.

    A row's decay is off by the roundings of its exponent (A log2 e, the product, the sums of dt over the 16 rows of a
    tile and the up to 24 tiles of a segment: 44 |dt A|) and by 8 (the exponential to 2^-22, products, slack), its input
    dt x B by 4, its sum by 2; y by 20 for 16 products and their sum, and by the gate's exponential and reciprocal."""
    h = E = H = torch.zeros(A.shape, dtype=A.dtype, device=A.device)
    ys, offs = [], []
    gate = z * torch.sigmoid(z)
    for t in range(x.shape[0]):
        v = dt[t][:, None] * A
        a, w = torch.exp(v), (dt[t] * x[t])[:, None] * B[t]
        h, size = a * h + w, a * H + w.abs()
        E = a * (E + (44 * v.abs() + 8) * ULP * H) + 4 * ULP * w.abs() + 2 * ULP * size
        H = size
        p = (h * C[t]).sum(-1) + D * x[t]
        m = (H * C[t].abs()).sum(-1) + (D * x[t]).abs()
        e = (E * C[t].abs()).sum(-1) + 20 * ULP * m
        ys.append(p * gate[t])
        offs.append((e + (2 * z[t].abs() + 10) * ULP * m) * gate[t].abs())
    return torch.stack(ys), torch.stack(offs), h, E


@pytest.mark.parametrize("length", [60, 1100, 16384])
def test_scan_within_the_bounds_of_32_bits(length):
    """Whole and cut sequences in fp32, up to a prompt of 16384 rows."""
    from sparseflow_b200.Kernels.selective_scan import selective_scan
    m = _scan_inputs((1, length), 64, 16, seed=length)
    m["dt"], m["dt_bias"] = m["dt"].abs() * 0.1, None
    y, f = selective_scan(**m, dt_softplus=False, return_final_state=True)
    rows = [m[k][0].double() for k in ("x", "dt", "B", "C", "z")]
    want, off, h, E = _scan_with_bounds(rows[0], rows[1], m["A"].double(), rows[2], rows[3], m["D"].double(), rows[4])
    assert ((y[0].double() - want).abs() <= off + ULP * want.abs()).all()
    assert ((f[0].double() - h).abs() <= E).all()


def test_scan_gradients_within_the_norm_of_32_bits():
    """Gradients of a cut sequence in fp32: a state remembers about 1 / |dt A| <= 20 rows here, so that each of the two
    chains that a gradient multiplies is off by at most 44 + 8 * 20 roundings."""
    from sparseflow_b200.Kernels.selective_scan import selective_scan
    m = _scan_inputs((1, 1100), 24, 16, seed=3)
    m["dt"], m["dt_bias"], m["A"] = 0.1 + m["dt"].abs() * 0.1, None, -0.5 - torch.rand(24, 16, device="cuda")
    names = ("x", "dt", "A", "B", "C", "D", "z")
    leaves = [m[k].requires_grad_() for k in names]
    dy = torch.randn_like(m["x"])
    got = torch.autograd.grad(selective_scan(**m, dt_softplus=False), leaves, dy)
    want = ref.scan(*ref.f64(*leaves), None, False, None, None, ref.f64(dy))
    for k, g in zip(names, got):
        off = (g.double().cpu() - want["d" + k]).norm() / want["d" + k].norm()
        assert off <= 2 * (44 + 8 * 20) * ULP, (k, off)


class _Guarded:
    """Buffers whose middle is handed out, to see afterwards that what lies around it has stayed."""

    def __init__(self):
        self.buffers = []

    def __call__(self, numel, dtype=torch.float32, pad=512):
        buf = torch.full((numel + 2 * pad,), -77.0, device="cuda").to(dtype)
        self.buffers.append((buf, pad))
        return buf.data_ptr() + pad * buf.element_size()

    def check(self):
        for i, (buf, pad) in enumerate(self.buffers):
            assert (buf[:pad] == -77).all() and (buf[-pad:] == -77).all(), i


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("length, dim, n, groups", [(1, 5, 3, 1), (17, 70, 13, 2), (700, 66, 16, 1), (33, 64, 40, 4)])
def test_scan_writes_its_outputs_alone(dtype, length, dim, n, groups):
    from sparseflow_b200 import _lib
    lib, s, give = _lib.load(), 2, _Guarded()
    m = _scan_inputs((s, length), dim, n, groups, dtype)
    init, df, dy = torch.randn(s, dim, n, device="cuda"), torch.randn(s, dim, n, device="cuda"), torch.randn_like(m["x"])
    p = {k: t.data_ptr() for k, t in m.items()}
    row, bc = (length * dim, dim), (length * groups * n, groups * n)
    d = ctypes.byref(_lib.SelectiveScanDesc(length, *row * 3, *bc * 2, s, dim, n, groups, 1, _lib.sf_dtype(dtype), 0))
    stream = torch.cuda.current_stream().cuda_stream
    ck = give(lib.sf_selective_scan_checkpoint_bytes(d) // 4)
    size = lib.sf_selective_scan_workspace_size(d)
    assert lib.sf_selective_scan(p["x"], p["dt"], p["A"], p["B"], p["C"], p["D"], p["z"], p["dt_bias"], init.data_ptr(),
                                 None, give(s * length * dim, dtype), give(s * dim * n), ck, d, give(size // 4), size,
                                 stream) == _lib.SF_OK
    size = lib.sf_selective_scan_backward_workspace_size(d)
    x, bc = s * length * dim, s * length * groups * n
    assert lib.sf_selective_scan_backward(
        p["x"], p["dt"], p["A"], p["B"], p["C"], p["D"], p["z"], p["dt_bias"], None, ck, dy.data_ptr(), df.data_ptr(),
        give(x, dtype), give(x, dtype), give(dim * n), give(bc, dtype), give(bc, dtype), give(dim), give(x, dtype),
        give(dim), give(s * dim * n), d, give(size // 4), size, stream) == _lib.SF_OK
    give.check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, per, dim", [(1, 1, 7), (6, 3, 96), (40, 20, 4104), (300, 1, 1000)])
def test_norm_writes_its_outputs_alone(dtype, rows, per, dim):
    from sparseflow_b200 import _lib
    lib, give, k = _lib.load(), _Guarded(), _lib.sf_dtype(dtype)
    y, res, dr, dx = (torch.randn(rows, dim, device="cuda").to(dtype) for _ in range(4))
    gate = torch.randn(rows // per, dim, device="cuda").to(dtype)
    w = [torch.randn(dim, device="cuda").to(dtype) for _ in range(3)]
    d = ctypes.byref(_lib.BlockNormDesc(rows, dim, dim, dim, per, dim, k, k, k, _lib.SF_GATE_SILU, 1.0, 1e-6))
    stream = torch.cuda.current_stream().cuda_stream
    inputs = [t.data_ptr() for t in (y, res, gate, *w)]
    rstd = torch.zeros(2 * rows, device="cuda")
    assert lib.sf_block_norm(*inputs, give(rows * dim, dtype), give(rows * dim, dtype), rstd.data_ptr(), d,
                             stream) == _lib.SF_OK
    size = lib.sf_block_norm_backward_workspace_size(d)
    assert lib.sf_block_norm_backward(*inputs, rstd.data_ptr(), dr.data_ptr(), dx.data_ptr(), give(rows * dim, dtype),
                                      give(rows * dim, dtype), give(rows // per * dim, dtype),
                                      *(give(dim, dtype) for _ in range(3)), d, give(size // 4), size,
                                      stream) == _lib.SF_OK
    give.check()
