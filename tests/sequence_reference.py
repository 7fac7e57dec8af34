"""The sequence operators in 64 bits, row by row from their formulas, for tests.

Every function takes ``mag``: with it, each term of each sum enters with its magnitude, so the result bounds what the
rounding errors of the sums can be relative to. ``close`` compares a kernel's output with the value:

    |got - ref| <= half an ulp of the output's type * |ref| + roundings * 2^-24 * magnitude

where `roundings` counts the fp32 roundings that an output can pass through, one after another.
"""
import torch

HALF_ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
# The smallest normal of a type, and half the spacing below it: results that underflow are off by an absolute amount.
TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}


def close(got, ref, mag, roundings, what=""):
    got_type = got.dtype
    got = got.detach().double().cpu()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    if not got.numel():
        return
    off = (got - ref).abs()
    bound = HALF_ULP[got_type] * 1.01 * ref.abs() + roundings * 2.0 ** -24 * mag + TINY[got_type]
    assert torch.isfinite(got).all(), what
    worst = (off / bound.clamp(min=1e-300)).max().item()
    assert worst <= 1.0, f"{what}: {worst:.2f} times the bound"


def f64(*tensors):
    out = [None if t is None else t.detach().double().cpu() for t in tensors]
    return out[0] if len(out) == 1 else out


def silu(v, mag=False):
    r = v * torch.sigmoid(v)
    return r.abs() if mag else r


def dsilu(v, mag=False):
    s = torch.sigmoid(v)
    return s * (1 + (v.abs() if mag else v) * (1 - s))


def _abs(mag, *ts):
    return [None if t is None else (t.abs() if mag else t) for t in ts]


def _edges(x, offsets):
    """(rows of x as [total, ...], list of (begin, end))."""
    if offsets is None:
        b, n = x.shape[:2]
        return [(i * n, (i + 1) * n) for i in range(b)]
    o = [int(v) for v in offsets]
    return list(zip(o, o[1:]))


def conv(x, weight, bias, act, init, offsets, dy=None, dfinal=None, mag=False):
    """(y, final, dx, dw, db, dinit) in 64 bits; the last four None without dy."""
    shape, (dim, w) = x.shape, weight.shape
    edges = _edges(x, offsets)
    xs = x.reshape(-1, dim)
    init = torch.zeros(len(edges), w - 1, dim, dtype=xs.dtype) if init is None else init
    bias = torch.zeros(dim, dtype=xs.dtype) if bias is None else bias
    ax, aw, ab, ai, ady, adf = _abs(mag, xs, weight, bias, init, dy, dfinal)
    y, final = torch.zeros_like(xs), torch.zeros_like(init)
    dx, dw, db, dinit = torch.zeros_like(xs), torch.zeros_like(weight), torch.zeros_like(bias), torch.zeros_like(init)
    ady = None if ady is None else ady.reshape(-1, dim)
    for s, (a, b) in enumerate(edges):
        n = b - a
        rows, arows = torch.cat([init[s], xs[a:b]]), torch.cat([ai[s], ax[a:b]])
        pre = bias + sum(weight[:, k] * rows[k: k + n] for k in range(w)) if n else rows[:0]
        size = ab + sum(aw[:, k] * arows[k: k + n] for k in range(w)) if n else rows[:0]
        # |silu'| <= 1.1, and the exponential in it is off by a few ulp of its own: |silu| counts too.
        y[a:b] = ((1.1 * size + silu(pre, True)) if mag else silu(pre)) if act else (size if mag else pre)
        final[s] = arows[n:] if mag else rows[n:]
        if dy is None:
            continue
        # silu'' <= 1/2: an error of pre reaches g by that much.
        g = ady[a:b] * ((dsilu(pre, True) + 0.5 * size + 1) if mag else dsilu(pre)) if act else ady[a:b]
        drows = torch.zeros_like(rows)
        for k in range(w):
            drows[k: k + n] += aw[:, k] * g
            dw[:, k] += (g * arows[k: k + n]).sum(0)
        db += g.sum(0)
        if adf is not None:
            drows[n:] += adf[s]
        dinit[s], dx[a:b] = drows[: w - 1], drows[w - 1:]
    out = (y.reshape(shape), final)
    return (*out, None, None, None, None) if dy is None else (*out, dx.reshape(shape), dw, db, dinit)


def scan(x, dt, A, B, C, D, z, bias, softplus, init, offsets, dy=None, dfinal=None, mag=False):
    """dict of y, final and, with dy, the gradients, in 64 bits. B, C [.., groups, state]."""
    shape, (dim, n), groups = x.shape, A.shape, B.shape[-2]
    per = dim // groups
    edges = _edges(x, offsets)
    flat = [t.reshape(-1, dim) if t is not None else None for t in (x, dt, z, dy)]
    x, dt, z, dy = flat
    wide = [t.reshape(-1, groups, n).repeat_interleave(per, 1) for t in (B, C)]  # [rows, dim, n]
    raw = dt if bias is None else dt + bias
    dt = torch.nn.functional.softplus(raw, threshold=1e9) if softplus else raw
    init = torch.zeros(len(edges), dim, n, dtype=x.dtype) if init is None else init
    D = torch.zeros(dim, dtype=x.dtype) if D is None else D
    decay = torch.exp(dt[..., None] * A)  # magnitudes too decay by this
    ax, Bw, Cw, aD, ai, ady, adf, adt, aA = _abs(mag, x, *wide, D, init, dy, dfinal, dt, A)
    gate = torch.ones_like(x) if z is None else silu(z, mag)
    h, p = torch.zeros(x.shape[0], dim, n, dtype=x.dtype), torch.zeros_like(x)
    hprev = torch.zeros_like(h)
    final = torch.zeros_like(init)
    for s, (a, b) in enumerate(edges):
        cur = ai[s]
        for t in range(a, b):
            hprev[t] = cur
            cur = decay[t] * cur + (adt[t] * ax[t])[:, None] * Bw[t]
            h[t] = cur
        final[s] = cur
    p = (h * Cw).sum(-1) + aD * ax
    out = {"y": (p * gate).reshape(shape), "final": final}
    if dy is None:
        return out
    gp = ady * gate
    gh, gall, ginit = torch.zeros(dim, n, dtype=x.dtype), torch.zeros_like(h), torch.zeros_like(init)
    for s, (a, b) in enumerate(edges):
        gh = torch.zeros(dim, n, dtype=x.dtype) if adf is None else adf[s].clone()
        for t in range(b - 1, a - 1, -1):
            gh = gh + gp[t][:, None] * Cw[t]
            gall[t] = gh
            gh = gh * decay[t]
        ginit[s] = gh
    q = gall * hprev * decay
    S = (gall * Bw).sum(-1)
    sp = torch.sigmoid(raw) if softplus else torch.ones_like(raw)
    ddt = (ax * S + (q * aA).sum(-1)) * sp
    lead = B.shape
    out.update(
        dx=(adt * S + aD * gp).reshape(shape), ddt=ddt.reshape(shape), dA=(q * adt[..., None]).sum(0),
        dB=(gall * (adt * ax)[..., None]).reshape(-1, groups, per, n).sum(2).reshape(lead),
        dC=(gp[..., None] * h).reshape(-1, groups, per, n).sum(2).reshape(lead),
        dD=(gp * ax).sum(0), dbias=ddt.sum(0), dinit=ginit,
        dz=None if z is None else (ady * p * dsilu(z, mag)).reshape(shape))
    return out


def norm(y, residual, gate, kind, w_post, w_pre, scale, alpha, eps, dr=None, dx=None, mag=False):
    """dict of r, x and, with dr or dx, the gradients, in 64 bits; gate broadcasts against y."""
    one = torch.ones(y.shape[-1], dtype=y.dtype)
    ws, wp, wq = (one if t is None else t for t in (scale, w_post, w_pre))
    r1 = ((y * y).mean(-1, keepdim=True) + eps).rsqrt() if w_post is not None else torch.ones_like(y[..., :1])
    sig = None if gate is None else torch.sigmoid(gate)
    act, dact = {None: (torch.ones_like(y), None), "linear": (gate, None if gate is None else torch.ones_like(gate)),
                 "silu": (None if gate is None else gate * sig, None if gate is None else dsilu(gate, mag)),
                 "sigmoid": (sig, None if gate is None else sig * (1 - sig))}[kind]
    res = torch.zeros_like(y) if residual is None else residual
    yh = y * r1
    r = alpha * res + ws * act * wp * yh
    r2 = ((r * r).mean(-1, keepdim=True) + eps).rsqrt() if w_pre is not None else torch.zeros_like(y[..., :1])
    ay, ares, aact, adact, aws, awp, awq, ayh, adr, adx = _abs(mag, y, res, act, dact, ws, wp, wq, yh, dr, dx)
    ar = abs(alpha) * ares + aws * aact * awp * ayh if mag else r
    # An error of one element of r' moves the whole row's rms: its share is bounded by the row's largest.
    rh = (ar + ar.square().mean(-1, keepdim=True).sqrt()) * r2 if mag else r * r2
    out = {"r": ar, "x": awq * rh}
    if dr is None and dx is None:
        return out
    dr = torch.zeros_like(y) if adr is None else adr
    dx = torch.zeros_like(y) if adx is None else adx
    sign = 1 if mag else -1
    q = awq * dx
    tot = dr + r2 * (q + sign * rh * (q * rh).mean(-1, keepdim=True))
    u = awp * ayh
    du = tot * aws * aact
    v = awp * du
    e = (tot * aact * u)
    out.update(dres=abs(alpha) * tot if mag else alpha * tot,
               dy=r1 * (v + sign * ayh * (v * ayh).mean(-1, keepdim=True)) if w_post is not None else v,
               dscale=e.flatten(0, -2).sum(0), dpost=(du * ayh).flatten(0, -2).sum(0),
               dpre=(dx * rh).flatten(0, -2).sum(0))
    if w_post is None:
        out["dy"] = du
    if gate is not None:
        g = tot * aws * u * adact
        out["dgate"] = g.sum(-2, keepdim=True) if gate.shape != y.shape else g
    return out
