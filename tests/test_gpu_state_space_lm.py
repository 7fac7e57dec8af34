"""The sequence operators together, as a language model uses them."""
import pytest
import torch

import sequence_reference as ref

pytestmark = pytest.mark.gpu


def _model(spiking=False, dtype=torch.float32, **kw):
    from sparseflow_b200.snn import SpikingStateSpaceLM
    torch.manual_seed(3)
    m = SpikingStateSpaceLM(40, 48, 2, spiking=spiking, v_threshold=0.1, **kw).cuda()
    for norm in m.norms:  # not all ones
        for p in norm.parameters():
            p.data += 0.1 * torch.randn_like(p)
    if dtype != torch.float32:
        m = m.to(dtype)
        for mixer in m.mixers:
            mixer.A_log.data = mixer.A_log.data.float()
    return m


def _plain(m, tokens):
    """The model's logits in 64 bits from the formulas (not spiking)."""
    f = ref.f64
    x = f(m.embedding.weight)[tokens.cpu()]
    n = ref.norm(x, None, None, None, None, f(m.first_weight), None, 1.0, 1e-6)
    res, x = n["r"], n["x"]
    for mixer, gate, norm in zip(m.mixers, m.gates, m.norms):
        a, z = (x @ f(mixer.in_proj.weight).T).split(mixer.inner, -1)
        a = ref.conv(a, *f(mixer.conv_weight, mixer.conv_bias), True, None, None)[0]
        p = a @ f(mixer.x_proj.weight).T
        k = mixer.groups * mixer.state
        B, C = (p[..., mixer.dt_rank + i * k: mixer.dt_rank + (i + 1) * k].unflatten(-1, (mixer.groups, mixer.state))
                for i in (0, 1))
        dt = p[..., : mixer.dt_rank] @ f(mixer.dt_proj.weight).T
        y = ref.scan(a, dt, -torch.exp(f(mixer.A_log)), B, C, f(mixer.D), z, f(mixer.dt_bias), True, None, None)["y"]
        g = x @ f(gate.weight).T + f(gate.bias)
        n = ref.norm(y @ f(mixer.out_proj.weight).T + f(mixer.out_proj.bias), res, g, "silu", *f(norm.post_weight, norm.pre_weight, norm.scale),
                     1.0, 1e-6)
        res, x = n["r"], n["x"]
    return x @ f(m.head.weight).T


@pytest.fixture(autouse=True)
def _exact_matmuls():
    old = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    yield
    torch.backends.cuda.matmul.allow_tf32 = old


@pytest.mark.parametrize("groups", [1, 2])
def test_logits_equal_the_formulas(groups):
    m = _model(groups=groups)
    tokens = torch.randint(0, 40, (2, 37), device="cuda")
    with torch.no_grad():
        got = m(tokens)
    want = _plain(m, tokens)
    # Two blocks of about 10 operators in fp32; the norms keep values of order 1.
    assert (got.double().cpu() - want).norm() <= 1e-5 * want.norm()


def test_prompt_and_steps_equal_the_whole():
    m = _model()
    tokens = torch.randint(0, 40, (3, 30), device="cuda")
    with torch.no_grad():
        whole = m(tokens)
        logits, states = m.prefill(tokens[:, :21])
        parts = [logits] + [m.step(tokens[:, t], states)[:, None] for t in range(21, 30)]
    assert (torch.cat(parts, 1) - whole).norm() <= 1e-5 * whole.norm()


def test_packed_sequences_equal_each_alone():
    m = _model()
    lengths = [5, 0, 17, 1]
    tokens = torch.randint(0, 40, (sum(lengths),), device="cuda")
    off = torch.tensor([0, 5, 5, 22, 23], dtype=torch.int32, device="cuda")
    with torch.no_grad():
        got = m(tokens, off)
        for a, b in zip(off.tolist(), off.tolist()[1:]):
            if b > a:
                alone = m(tokens[None, a:b])[0]
                assert (got[a:b] - alone).norm() <= 1e-5 * alone.norm()


def test_spiking_prompt_and_steps():
    """Spikes and event-driven projections: the prompt token by token. A membrane within rounding of the threshold may
    fire in one and not in the other, so a few logits in a hundred may differ, and none does before such a spike."""
    from sparseflow_b200.Ops.lif_node import reset_net
    m = _model(spiking=True).eval()
    tokens = torch.randint(0, 40, (2, 24), device="cuda")
    with torch.no_grad():
        whole = m(tokens)
        rate = m.mixers[0].lif.v.abs().max()
        assert torch.isfinite(whole).all() and rate > 0
        reset_net(m)
        _, states = m.prefill(tokens[:, :10])
        parts = [m.step(tokens[:, t], states) for t in range(10, 24)]
    got = torch.stack(parts, 1)
    off = (got - whole[:, 10:]).norm(dim=-1) > 1e-4 * whole[:, 10:].norm(dim=-1)
    assert off.float().mean() <= 0.3


def test_spiking_mixer_refuses_training_and_packing():
    m = _model(spiking=True)
    tokens = torch.randint(0, 40, (2, 5), device="cuda")
    with pytest.raises(RuntimeError, match="gradient"):
        m(tokens)
    with pytest.raises(ValueError, match="spiking"):
        m.eval()(tokens.flatten(), torch.tensor([0, 5, 10], dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_training_learns(dtype):
    """A sequence whose next token follows from the last two: the loss falls well below that of guessing."""
    m = _model(dtype=dtype)
    opt = torch.optim.Adam(m.parameters(), lr=1e-2)
    g = torch.Generator(device="cuda").manual_seed(0)
    first = None
    for _ in range(60):
        t = torch.randint(0, 8, (8, 34), device="cuda", generator=g)
        for k in range(2, 34):
            t[:, k] = (t[:, k - 1] + t[:, k - 2]) % 8
        loss = torch.nn.functional.cross_entropy(m(t[:, :-1]).float().flatten(0, 1), t[:, 1:].flatten())
        opt.zero_grad()
        loss.backward()
        assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in m.parameters() if p.requires_grad)
        opt.step()
        first = loss.item() if first is None else first
    assert loss.item() < 0.5 * first
