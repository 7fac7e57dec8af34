"""Cases of the sequence operators: the short causal convolution, the selective state space scan (each for prompts,
for training and for single tokens) and the norms around a block with their gate and residual scale.

A case is one call as a program makes it. ``run`` makes it in plain torch operations in 32 bits, or, where ``own`` is
true, through the package's public functions."""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # One user, one token: the latency of a decoding step.
        {"name": "conv_token_1", "op": "conv_step", "rows": 1, "dim": 2048, "width": 4, "dtype": "bf16"},
        # A serving batch of 200 requests whose states lie scattered in a pool.
        {"name": "conv_token_200", "op": "conv_step", "rows": 200, "dim": 5120, "width": 4, "dtype": "bf16"},
        # Ragged prompts packed in one call, continuing from cached states; one is empty, one has a single token.
        {"name": "conv_prompt_ragged", "op": "conv", "seqs": 9, "tokens": 5003, "dim": 4096, "width": 4,
         "dtype": "bf16", "ragged": True, "train": False},
        # A training step's layer.
        {"name": "conv_train", "op": "conv", "seqs": 8, "tokens": 16384, "dim": 4096, "width": 4, "dtype": "bf16",
         "ragged": False, "train": True},
        # One user, one token.
        {"name": "scan_token_1", "op": "scan_step", "rows": 1, "dim": 2048, "groups": 1, "state": 16, "dtype": "bf16"},
        # A serving batch of 256 requests, states in a pool.
        {"name": "scan_token_256", "op": "scan_step", "rows": 256, "dim": 5120, "groups": 1, "state": 16,
         "dtype": "bf16"},
        # One long prompt: few rows side by side, a long way to go.
        {"name": "scan_prompt_long", "op": "scan", "seqs": 1, "tokens": 16384, "dim": 2048, "groups": 1, "state": 16,
         "dtype": "f16", "ragged": False, "train": False},
        # Ragged prompts packed in one call, continuing from cached states.
        {"name": "scan_prompt_ragged", "op": "scan", "seqs": 9, "tokens": 5003, "dim": 4096, "groups": 1, "state": 16,
         "dtype": "bf16", "ragged": True, "train": False},
        # A training step's layer.
        {"name": "scan_train", "op": "scan", "seqs": 4, "tokens": 8192, "dim": 4096, "groups": 1, "state": 16,
         "dtype": "bf16", "ragged": False, "train": True},
        # A small model trained in 32 bits, with odd sizes and two groups.
        {"name": "scan_train_odd", "op": "scan", "seqs": 3, "tokens": 1503, "dim": 770, "groups": 2, "state": 13,
         "dtype": "f32", "ragged": False, "train": True},
        # The norms around a block in a decoding step of eight requests.
        {"name": "norm_token_8", "op": "norm", "seqs": 8, "tokens": 8, "dim": 2048, "dtype": "bf16",
         "residual": "bf16", "gate": "rows", "train": False},
        # A training step's layer, with the residual stream in 32 bits.
        {"name": "norm_train", "op": "norm", "seqs": 4, "tokens": 8192, "dim": 4096, "dtype": "bf16",
         "residual": "f32", "gate": "rows", "train": True},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, spread over the logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["conv", "conv", "conv_step", "scan", "scan", "scan", "scan_step", "norm", "norm"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    # Widths of layers: any number, or a multiple of 64 as most models have.
    dim = _spread(rng, 64, 8192)
    if rng.random() < 0.6:
        dim = max(64, dim // 64 * 64)
    if dim == 3 * 1024:
        dim += 64
    if op == "conv_step":
        return {"op": op, "rows": _spread(rng, 1, 512), "dim": dim, "width": rng.choice([2, 3, 4, 4, 6]),
                "dtype": dtype}
    groups = rng.choice([1, 1, 1, 2, 4])
    state = rng.choice([16, 16, 16, 8, 32, rng.randint(1, 64)])
    if op == "scan_step":
        rows = _spread(rng, 1, min(512, max(1, (100 << 20) // (dim * state))))
        return {"op": op, "rows": rows, "dim": dim // groups * groups, "groups": groups, "state": state,
                "dtype": dtype}
    train = rng.random() < 0.5
    seqs = _spread(rng, 1, 16)
    most = 8192 * 4096 // (2 if dtype == "f32" else 1)  # rows times channels, so that a case in 32 bits costs no more
    if op == "norm":
        tokens = _spread(rng, 1, most // dim)
        return {"op": op, "seqs": seqs, "tokens": max(1, tokens // seqs) * seqs, "dim": dim, "dtype": dtype,
                "residual": rng.choice([dtype, "f32"]), "gate": rng.choice(["rows", "sequence", "none"]),
                "train": train}
    ragged = not train and rng.random() < 0.5
    if op == "conv":
        tokens = _spread(rng, 16, most // dim)
        case = {"op": op, "seqs": seqs, "tokens": tokens, "dim": dim, "width": rng.choice([2, 3, 4, 4, 6])}
    else:
        dim = dim // groups * groups
        tokens = _spread(rng, 16, min(32768, most * 16 // (dim * max(16, state))))
        case = {"op": op, "seqs": seqs, "tokens": tokens, "dim": dim, "groups": groups, "state": state}
    if not ragged:
        case["tokens"] = max(1, tokens // seqs) * seqs
    return {**case, "dtype": dtype, "ragged": ragged, "train": train}


# ---------------------------------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------------------------------

def _lengths(case, seed):
    """Lengths of the packed sequences: random cuts of the total; with four or more, one of 0 and one of 1 token."""
    n, total = case["seqs"], case["tokens"]
    g = torch.Generator().manual_seed(seed)
    if n < 4 or total < 4:
        cuts = torch.sort(torch.randint(0, total + 1, (n - 1,), generator=g)).values.tolist()
        edges = [0] + cuts + [total]
        return [b - a for a, b in zip(edges, edges[1:])]
    share = torch.rand(n - 2, generator=g) + 0.1
    rest = (share / share.sum() * (total - 1)).long().tolist()
    rest[0] += total - 1 - sum(rest)
    return rest[:1] + [0] + rest[1:] + [1]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    f32 = torch.float32

    def normal(*shape, dtype=dt, scale=1.0, shift=0.0):
        return (torch.randn(*shape, device="cuda", generator=g) * scale + shift).to(dtype)

    op, dim = case["op"], case["dim"]
    s = {"case": case}
    if op in ("conv", "conv_step"):
        # Weights as a layer of this fan-in is initialised.
        w = case["width"]
        s["weight"] = normal(dim, w, scale=w ** -0.5)
        s["bias"] = normal(dim, scale=0.1)
    elif op in ("scan", "scan_step"):
        n, groups = case["state"], case["groups"]
        # Decays of a trained layer: near -1 .. -n, each moved; steps between about 0.001 and 0.1.
        s["A"] = -(torch.arange(1, n + 1, device="cuda", dtype=f32) * torch.exp(normal(dim, n, dtype=f32, scale=0.3)))
        step = torch.exp(torch.rand(dim, device="cuda", generator=g) * math.log(100.0) + math.log(1e-3))
        s["dt_bias"] = step + torch.log(-torch.expm1(-step))
        s["D"] = normal(dim, dtype=f32, scale=0.1, shift=1.0)
    if op in ("conv_step", "scan_step"):
        rows = case["rows"]
        pool = rows + rows // 8 + 1
        s["slots"] = torch.randperm(pool, device="cuda", generator=g)[:rows].to(torch.int32)
        s["x"] = normal(rows, dim)
        if op == "conv_step":
            s["pool"] = normal(pool, case["width"] - 1, dim)
        else:
            s["dt"], s["z"] = normal(rows, dim, scale=0.5), normal(rows, dim)
            s["B"], s["C"] = normal(rows, groups, n), normal(rows, groups, n)
            s["pool"] = normal(pool, dim, n, dtype=f32, scale=0.3)
        return s
    seqs, total = case["seqs"], case["tokens"]
    if op == "norm":
        shape = (seqs, total // seqs, dim)
        s["y"] = normal(*shape)
        s["residual"] = normal(*shape, dtype=DTYPES[case["residual"]], scale=2.0)
        s["gate"] = {"rows": shape, "sequence": (seqs, 1, dim), "none": None}[case["gate"]]
        if s["gate"] is not None:
            s["gate"] = normal(*s["gate"])
        for name in ("post_weight", "pre_weight"):
            s[name] = normal(dim, dtype=f32, scale=0.2, shift=1.0)
        s["scale"] = normal(dim, dtype=f32, scale=0.1, shift=0.5)
        leaves = ["y", "residual", "gate", "post_weight", "pre_weight", "scale"]
        if case["train"]:
            s["grad_residual"] = normal(*shape, dtype=DTYPES[case["residual"]])
            s["grad_normed"] = normal(*shape)
    else:
        if case["ragged"]:
            shape = (total,)
            lengths = torch.tensor([0] + _lengths(case, seed)).cumsum(0)
            s["offsets"] = lengths.to(device="cuda", dtype=torch.int32)
        else:
            shape = (seqs, total // seqs)
        s["x"] = normal(*shape, dim)
        if op == "conv":
            if case["ragged"]:
                s["state"] = normal(seqs, case["width"] - 1, dim)
            leaves = ["x", "weight", "bias"]
        else:
            s["x"] = torch.nn.functional.silu(s["x"].float()).to(dt)  # what the convolution before it gives
            s["dt"], s["z"] = normal(*shape, dim, scale=0.5), normal(*shape, dim)
            s["B"], s["C"] = normal(*shape, groups, n), normal(*shape, groups, n)
            if case["ragged"]:
                s["state"] = normal(seqs, dim, n, dtype=f32, scale=0.3)
            leaves = ["x", "dt", "A", "B", "C", "D", "z", "dt_bias"]
        if case["train"]:
            s["grad"] = normal(*shape, dim)
    if case["train"]:
        s["leaves"] = [k for k in leaves if s[k] is not None]
        for k in s["leaves"]:
            s[k].requires_grad_()
    return s


# ---------------------------------------------------------------------------------------------------------------------
# The package's functions
# ---------------------------------------------------------------------------------------------------------------------

def _own_conv(s):
    from sparseflow_b200.Kernels.causal_conv1d import causal_conv1d
    if not s["case"]["train"]:
        y, state = causal_conv1d(s["x"], s["weight"], s["bias"], activation="silu", initial_state=s.get("state"),
                                 seq_offsets=s.get("offsets"), return_final_state=True)
        return {"y": y, "state": state}
    y = causal_conv1d(s["x"], s["weight"], s["bias"], activation="silu")
    return {"y": y, "grads": torch.autograd.grad(y, [s[k] for k in s["leaves"]], s["grad"])}


def _own_conv_step(s):
    from sparseflow_b200.Kernels.causal_conv1d import causal_conv1d_update
    y = causal_conv1d_update(s["x"], s["pool"], s["weight"], s["bias"], activation="silu", state_indices=s["slots"])
    return {"y": y, "pool": s["pool"]}


def _own_scan(s):
    from sparseflow_b200.Kernels.selective_scan import selective_scan
    args = (s["x"], s["dt"], s["A"], s["B"], s["C"], s["D"], s["z"], s["dt_bias"])
    if not s["case"]["train"]:
        y, state = selective_scan(*args, initial_state=s.get("state"), seq_offsets=s.get("offsets"),
                                  return_final_state=True)
        return {"y": y, "state": state}
    y = selective_scan(*args)
    return {"y": y, "grads": torch.autograd.grad(y, [s[k] for k in s["leaves"]], s["grad"])}


def _own_scan_step(s):
    from sparseflow_b200.Kernels.selective_scan import selective_scan_update
    y = selective_scan_update(s["x"], s["dt"], s["A"], s["B"], s["C"], s["pool"], s["D"], s["z"], s["dt_bias"],
                              state_indices=s["slots"])
    return {"y": y, "pool": s["pool"]}


def _own_norm(s):
    from sparseflow_b200.Kernels.block_norm import block_norm
    residual, normed = block_norm(s["y"], s["residual"], s["post_weight"], s["pre_weight"], gate=s["gate"],
                                  gate_activation="silu", scale=s["scale"], eps=1e-6)
    out = {"residual": residual, "normed": normed}
    if s["case"]["train"]:
        out["grads"] = torch.autograd.grad((residual, normed), [s[k] for k in s["leaves"]],
                                           (s["grad_residual"], s["grad_normed"]))
    return out


# ---------------------------------------------------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------------------------------------------------

def _silu(v):
    return v / (1 + torch.exp(-v))


def _softplus(v):
    return torch.clamp(v, min=0) + torch.log1p(torch.exp(-v.abs()))


def _conv_rows(rows, weight, bias):
    """rows [..., L + W - 1, dim], the W - 1 rows before the first one included -> [..., L, dim]."""
    return _silu((rows.unfold(-2, weight.shape[1], 1) * weight).sum(-1) + bias)


def _plain_conv(s):
    case, dt = s["case"], s["x"].dtype
    w = case["width"]
    if case["train"]:
        leaves = [s[k].detach().float().requires_grad_() for k in s["leaves"]]
        x, weight, bias = leaves
        y = _conv_rows(torch.cat([torch.zeros_like(x[:, : w - 1]), x], 1) if x.shape[1] >= w - 1 else
                       torch.nn.functional.pad(x, (0, 0, w - 1, 0)), weight, bias)
        grads = torch.autograd.grad(y, leaves, s["grad"].float())
        return {"y": y.detach().to(dt), "grads": [g.to(s[k].dtype) for g, k in zip(grads, s["leaves"])]}
    weight, bias = s["weight"].float(), s["bias"].float()
    if not case["ragged"]:
        rows = torch.nn.functional.pad(s["x"].float(), (0, 0, w - 1, 0))
        return {"y": _conv_rows(rows, weight, bias).to(dt), "state": rows[:, -(w - 1):].to(dt)}
    x, state, offsets = s["x"].float(), s["state"].float(), s["offsets"].long()
    total, seqs = x.shape[0], state.shape[0]
    # Row t of sequence q is row t + (w - 1) (q + 1) of the states and sequences laid one after another.
    q = torch.searchsorted(offsets[1:], torch.arange(total, device=x.device), right=True)
    joined = x.new_empty(total + (w - 1) * seqs, x.shape[1])
    at = torch.arange(total, device=x.device) + (w - 1) * (q + 1)
    joined[at] = x
    first = offsets[:-1] + (w - 1) * torch.arange(seqs, device=x.device)
    tail = torch.arange(w - 1, device=x.device)
    joined[(first[:, None] + tail).reshape(-1)] = state.reshape(-1, x.shape[1])
    y = _conv_rows(joined, weight, bias)[at - (w - 1)]
    last = offsets[1:] + (w - 1) * torch.arange(seqs, device=x.device)
    return {"y": y.to(dt), "state": joined[last[:, None] + tail].to(dt)}


def _plain_conv_step(s):
    slots = s["slots"].long()
    rows = torch.cat([s["pool"][slots], s["x"][:, None]], 1)
    s["pool"][slots] = rows[:, 1:]
    return {"y": _conv_rows(rows.float(), s["weight"].float(), s["bias"].float())[:, 0].to(s["x"].dtype),
            "pool": s["pool"]}


def _recur(a, b):
    """h_t = a_t h_(t-1) + b_t along dim 1 from h = 0, by doubling the stretch that each entry covers."""
    reach = 1
    while reach < a.shape[1]:
        b = torch.cat([b[:, :reach], b[:, reach:] + a[:, reach:] * b[:, :-reach]], 1)
        a = torch.cat([a[:, :reach], a[:, reach:] * a[:, :-reach]], 1)
        reach *= 2
    return b


def _plain_scan(s):
    case, kind = s["case"], s["x"].dtype
    x, B, C, z = (s[k].detach().float() for k in ("x", "B", "C", "z"))
    A, D = s["A"].detach(), s["D"].detach()
    raw = s["dt"].detach().float() + s["dt_bias"].detach()
    if case["ragged"]:
        x, B, C, z, raw = (v[None] for v in (x, B, C, z, raw))
    per = case["dim"] // case["groups"]
    B, C = (v.repeat_interleave(per, 2) for v in (B, C))  # [.., L, dim, state]
    dt = _softplus(raw)
    a = torch.exp(dt[..., None] * A)
    b = (dt * x)[..., None] * B
    if case["ragged"]:
        offsets = s["offsets"].long()
        begins, some = offsets[:-1], offsets[1:] > offsets[:-1]
        at = torch.where(some, begins, x.shape[1])  # a row past the end takes the empty sequences' share
        carried = b.new_zeros(x.shape[1] + 1, *b.shape[2:])
        carried[at] = torch.exp(dt[0, begins.clamp(max=x.shape[1] - 1), :, None] * A) * s["state"]
        b = b + carried[:-1]
        start = torch.zeros(x.shape[1] + 1, 1, 1, dtype=torch.bool, device=x.device)
        start[at] = True
        h = _recur(a.masked_fill(start[:-1], 0.0), b)
        del a, b, carried
        state = torch.where(some[:, None, None], h[0, (offsets[1:] - 1).clamp(min=0)], s["state"])
    else:
        h = _recur(a, b)
        del b
        state = h[:, -1].contiguous()
    p = (C * h).sum(-1) + D * x
    sig = 1 / (1 + torch.exp(-z))
    y = (p * z * sig).to(kind)
    if not case["train"]:
        return {"y": y[0] if case["ragged"] else y, "state": state}
    gy = s["grad"].float()
    gp = gy * z * sig
    gz = gy * p * sig * (1 + z * (1 - sig))
    split = (x.shape[0], x.shape[1], case["groups"], per, case["state"])
    gC = (gp[..., None] * h).view(split).sum(3)
    later = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1).flip(1)
    gh = _recur(later, (gp[..., None] * C).flip(1)).flip(1)
    del later, C
    ga = gh * torch.cat([torch.zeros_like(h[:, :1]), h[:, :-1]], 1) * a
    del h, a
    gB = ((dt * x)[..., None] * gh).view(split).sum(3)
    inner = (gh * B).sum(-1)
    del gh, B
    gdt = (x * inner + (ga * A).sum(-1)) / (1 + torch.exp(-raw))
    grads = {"x": dt * inner + D * gp, "dt": gdt, "A": (ga * dt[..., None]).sum((0, 1)), "B": gB, "C": gC,
             "D": (gp * x).sum((0, 1)), "z": gz, "dt_bias": gdt.sum((0, 1))}
    return {"y": y, "grads": [grads[k].to(s[k].dtype) for k in s["leaves"]]}


def _plain_scan_step(s):
    case, slots = s["case"], s["slots"].long()
    x, z = s["x"].float(), s["z"].float()
    per = case["dim"] // case["groups"]
    B, C = (s[k].float().repeat_interleave(per, 1) for k in ("B", "C"))
    dt = _softplus(s["dt"].float() + s["dt_bias"])
    h = torch.exp(dt[..., None] * s["A"]) * s["pool"][slots] + (dt * x)[..., None] * B
    s["pool"][slots] = h
    y = ((h * C).sum(-1) + s["D"] * x) * _silu(z)
    return {"y": y.to(s["x"].dtype), "pool": s["pool"]}


def _rms(v):
    return v * torch.rsqrt((v * v).mean(-1, keepdim=True) + 1e-6)


def _plain_norm(s):
    train = s["case"]["train"]
    f = {k: None if s[k] is None else s[k].detach().float().requires_grad_(train)
         for k in ("y", "residual", "gate", "post_weight", "pre_weight", "scale")}
    v = _rms(f["y"]) * f["post_weight"] * f["scale"]
    if f["gate"] is not None:
        v = v * _silu(f["gate"])
    residual = f["residual"] + v
    normed = _rms(residual) * f["pre_weight"]
    out = {"residual": residual.detach().to(s["residual"].dtype), "normed": normed.detach().to(s["y"].dtype)}
    if train:
        grads = torch.autograd.grad((residual, normed), [f[k] for k in s["leaves"]],
                                    (s["grad_residual"].float(), s["grad_normed"].float()))
        out["grads"] = [g.to(s[k].dtype) for g, k in zip(grads, s["leaves"])]
    return out


def run(state):
    op = state["case"]["op"]
    if own:
        return {"conv": _own_conv, "conv_step": _own_conv_step, "scan": _own_scan, "scan_step": _own_scan_step,
                "norm": _own_norm}[op](state)
    return {"conv": _plain_conv, "conv_step": _plain_conv_step, "scan": _plain_scan, "scan_step": _plain_scan_step,
            "norm": _plain_norm}[op](state)


# ---------------------------------------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------

def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}
    e, op, dim = size[case["dtype"]], case["op"], case["dim"]
    if op == "conv_step":
        w, n = case["width"], case["rows"] * dim
        # x and y; the state's rows but the oldest kept one are read, and all written; weight and bias
        return {"bytes": e * (n * (2 + 2 * (w - 1)) + dim * (w + 1)), "flops": n * (2 * w + 5)}
    if op == "scan_step":
        n, k = case["rows"] * dim, case["state"]
        return {"bytes": e * (4 * n + 2 * case["rows"] * case["groups"] * k) + 8 * n * k + 4 * dim * (k + 2),
                "flops": n * (7 * k + 12)}
    n, seqs = case["tokens"] * dim, case["seqs"]
    if op == "norm":
        r = size[case["residual"]]
        gate = {"rows": n, "sequence": seqs * dim, "none": 0}[case["gate"]]
        moved = 2 * n * e + 2 * n * r + gate * e + 3 * 4 * dim
        if not case["train"]:
            return {"bytes": moved, "flops": 14 * n}
        # the backward pass reads the inputs and two gradients and writes the gradients of the inputs
        return {"bytes": moved + 3 * n * e + 3 * n * r + 2 * gate * e + 9 * 4 * dim, "flops": 50 * n}
    if op == "conv":
        w = case["width"]
        state = 2 * seqs * (w - 1) * dim if case["ragged"] else 0 if case["train"] else seqs * (w - 1) * dim
        if not case["train"]:
            return {"bytes": e * (2 * n + state + dim * (w + 1)), "flops": n * (2 * w + 5)}
        return {"bytes": e * (5 * n + 3 * dim * (w + 1)), "flops": n * (8 * w + 18)}
    k, bc = case["state"], 2 * case["tokens"] * case["groups"] * case["state"]
    state = 0 if case["train"] else 4 * seqs * dim * k * (2 if case["ragged"] else 1)
    if not case["train"]:
        return {"bytes": e * (4 * n + bc) + state + 4 * dim * (k + 2), "flops": n * (7 * k + 12)}
    # forward x, dt, z -> y; backward x, dt, z, gy -> gx, gdt, gz; B and C read twice, their gradients written
    return {"bytes": e * (11 * n + 3 * bc) + 3 * 4 * dim * (k + 2), "flops": n * (27 * k + 40)}


# ---------------------------------------------------------------------------------------------------------------------
# The definitions in 64 bits, step by step along the sequence
# ---------------------------------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    v = {k: t.detach().double() if torch.is_tensor(t) and t.is_floating_point() else t for k, t in s.items()}
    return {"conv": _exact_conv, "conv_step": _exact_conv_step, "scan": _exact_scan, "scan_step": _exact_scan_step,
            "norm": _exact_norm}[case["op"]](case, v)


def _sig(t):
    return torch.sigmoid(t)


def _exact_conv(case, v):
    w = case["width"]
    if not case["ragged"]:
        x, weight, bias = v["x"], v["weight"], v["bias"]
        seqs, length = x.shape[:2]
        pre = bias.expand_as(x).clone()
        for k in range(w):  # the tap that looks w - 1 - k rows back
            back = w - 1 - k
            if back < length:
                pre[:, back:] += weight[:, k] * x[:, : length - back]
        out = {"y": pre * _sig(pre)}
        if not case["train"]:
            state = x.new_zeros(seqs, w - 1, x.shape[2])
            keep = min(w - 1, length)
            state[:, w - 1 - keep:] = x[:, length - keep:]
            return {**out, "state": state}
        g = v["grad"] * _sig(pre) * (1 + pre * (1 - _sig(pre)))
        gx, gw = torch.zeros_like(x), torch.zeros_like(weight)
        for k in range(w):
            back = w - 1 - k
            if back < length:
                gx[:, : length - back] += weight[:, k] * g[:, back:]
                gw[:, k] = (g[:, back:] * x[:, : length - back]).sum((0, 1))
        return {**out, "grads": [gx, gw, g.sum((0, 1))]}
    ys, states = [], []
    edges = v["offsets"].tolist()
    for q, (a, b) in enumerate(zip(edges, edges[1:])):
        rows = torch.cat([v["state"][q], v["x"][a:b]])
        pre = v["bias"].expand(b - a, -1).clone()
        for k in range(w):
            pre += v["weight"][:, k] * rows[k: k + b - a]
        ys.append(pre * _sig(pre))
        states.append(rows[b - a:])
    return {"y": torch.cat(ys), "state": torch.stack(states)}


def _exact_conv_step(case, v):
    w, slots = case["width"], v["slots"].long()
    pre = v["bias"] + v["weight"][:, w - 1] * v["x"]
    pool = v["pool"].clone()
    for k in range(w - 1):
        pre = pre + v["weight"][:, k] * v["pool"][slots, k]
        pool[slots, k] = v["pool"][slots, k + 1] if k + 1 < w - 1 else v["x"]
    return {"y": pre * _sig(pre), "pool": pool}


def _wide(t, case):
    """[.., groups, state] -> [.., dim, state], each group's values for its channels."""
    per = case["dim"] // case["groups"]
    return t[..., :, None, :].expand(*t.shape[:-1], per, t.shape[-1]).reshape(*t.shape[:-2], case["dim"], t.shape[-1])


def _exact_scan(case, v):
    softplus = torch.nn.functional.softplus
    if case["ragged"]:
        y, states = torch.empty_like(v["x"]), []
        edges = v["offsets"].tolist()
        for q, (a, b) in enumerate(zip(edges, edges[1:])):
            h = v["state"][q]
            for t in range(a, b):
                dt = softplus(v["dt"][t] + v["dt_bias"], threshold=1e9)
                h = torch.exp(dt[:, None] * v["A"]) * h + (dt * v["x"][t])[:, None] * _wide(v["B"][t], case)
                y[t] = (h * _wide(v["C"][t], case)).sum(-1)
            states.append(h)
        return {"y": (y + v["D"] * v["x"]) * v["z"] * _sig(v["z"]), "state": torch.stack(states)}
    x, A, D, z = v["x"], v["A"], v["D"], v["z"]
    raw = v["dt"] + v["dt_bias"]
    dt = softplus(raw, threshold=1e9)
    length = x.shape[1]
    h = x.new_zeros(x.shape[0], case["dim"], case["state"])
    hs, p = [h], torch.empty_like(x)
    for t in range(length):
        h = torch.exp(dt[:, t, :, None] * A) * h + (dt[:, t] * x[:, t])[..., None] * _wide(v["B"][:, t], case)
        p[:, t] = (h * _wide(v["C"][:, t], case)).sum(-1)
        if case["train"]:
            hs.append(h)
    p += D * x
    s = _sig(z)
    out = {"y": p * z * s}
    if not case["train"]:
        return {**out, "state": h}
    gp = v["grad"] * z * s
    grads = {"z": v["grad"] * p * s * (1 + z * (1 - s)), "D": (gp * x).sum((0, 1)), "A": torch.zeros_like(A),
             "x": torch.empty_like(x), "dt": torch.empty_like(x), "B": torch.empty_like(v["B"]),
             "C": torch.empty_like(v["C"])}
    split = (x.shape[0], case["groups"], case["dim"] // case["groups"], case["state"])
    gh = torch.zeros_like(h)
    for t in range(length - 1, -1, -1):
        gpt, dtt, xt = gp[:, t, :, None], dt[:, t, :, None], x[:, t, :, None]
        gh = gh + gpt * _wide(v["C"][:, t], case)
        grads["C"][:, t] = (gpt * hs[t + 1]).view(split).sum(2)
        grads["B"][:, t] = (gh * dtt * xt).view(split).sum(2)
        inner = (gh * _wide(v["B"][:, t], case)).sum(-1)
        a = torch.exp(dtt * A)
        ga = gh * hs[t] * a
        grads["A"] += (ga * dtt).sum(0)
        grads["x"][:, t] = dt[:, t] * inner + D * gp[:, t]
        grads["dt"][:, t] = (x[:, t] * inner + (ga * A).sum(-1)) * _sig(raw[:, t])
        gh = a * gh
        hs.pop()
    grads["dt_bias"] = grads["dt"].sum((0, 1))
    return {**out, "grads": [grads[k] for k in v["leaves"]]}


def _exact_scan_step(case, v):
    slots = v["slots"].long()
    dt = torch.nn.functional.softplus(v["dt"] + v["dt_bias"], threshold=1e9)
    h = v["pool"][slots] * torch.exp(dt[..., None] * v["A"]) + (dt * v["x"])[..., None] * _wide(v["B"], case)
    pool = v["pool"].clone()
    pool[slots] = h
    y = (h * _wide(v["C"], case)).sum(-1) + v["D"] * v["x"]
    return {"y": y * v["z"] * _sig(v["z"]), "pool": pool}


def _exact_norm(case, v):
    y, w1, w2, scale, dim = v["y"], v["post_weight"], v["pre_weight"], v["scale"], case["dim"]
    r1 = ((y ** 2).sum(-1, keepdim=True) / dim + 1e-6) ** -0.5
    z = v["gate"]
    s = None if z is None else _sig(z)
    gate = torch.ones_like(y) if z is None else (z * s).expand_as(y)
    unit = y * r1
    res = v["residual"] + scale * gate * w1 * unit
    r2 = ((res ** 2).sum(-1, keepdim=True) / dim + 1e-6) ** -0.5
    out = {"residual": res, "normed": res * r2 * w2}
    if not case["train"]:
        return out
    gn = v["grad_normed"]
    hat = res * r2
    total = v["grad_residual"] + r2 * (w2 * gn - hat * (w2 * gn * hat).sum(-1, keepdim=True) / dim)
    gu = total * scale * gate
    grads = {"residual": total, "scale": (total * gate * unit * w1).sum((0, 1)),
             "post_weight": (gu * unit).sum((0, 1)), "pre_weight": (gn * hat).sum((0, 1)),
             "y": r1 * (w1 * gu - unit * (w1 * gu * unit).sum(-1, keepdim=True) / dim)}
    if z is not None:
        g = total * scale * unit * w1 * s * (1 + z * (1 - s))
        grads["gate"] = g.sum(1, keepdim=True) if case["gate"] == "sequence" else g
    return {**out, "grads": [grads[k] for k in v["leaves"]]}
