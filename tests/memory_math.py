"""Plain float64 restatements of the memory operators for their tests: numpy
and torch on the CPU, written from the formulas, step by step."""

import torch


def layer_norm(x, w, b, eps, dy=None):
    x = x.double()
    w = torch.ones(x.shape[-1], dtype=torch.float64) if w is None else w.double()
    b = torch.zeros(x.shape[-1], dtype=torch.float64) if b is None else b.double()
    mean = x.mean(-1, keepdim=True)
    sigma = ((x - mean) ** 2).mean(-1, keepdim=True).add(eps).sqrt()
    unit = (x - mean) / sigma
    y = unit * w + b
    if dy is None:
        return y
    g = dy.double() * w
    dx = (g - g.mean(-1, keepdim=True) - unit * (g * unit).mean(-1, keepdim=True)) / sigma
    return y, dx, (dy.double() * unit).sum(0), dy.double().sum(0)


def attention(q, k, v, decay, state, resets, scale, do=None, dlast=None):
    """(o, last) and, with do or dlast, (o, last, dq, dk, dv, dstate)."""
    T, E, H, Dk = q.shape
    Dv = v.shape[3]
    q, k, v, decay = q.double(), k.double(), v.double(), decay.double()
    S = torch.zeros(E, H, Dk, Dv, dtype=torch.float64) if state is None else state.double().clone()
    cut = torch.zeros(T, E, dtype=torch.bool) if resets is None else resets.bool()
    o, states = torch.zeros(T, E, H, Dv, dtype=torch.float64), []
    for t in range(T):
        S = torch.where(cut[t][:, None, None, None], torch.zeros_like(S), S) * decay[None, :, None, None]
        S = S + torch.einsum("ehi,ehj->ehij", k[t], v[t])
        o[t] = scale * torch.einsum("ehi,ehij->ehj", q[t], S)
        states.append(S)
    if do is None and dlast is None:
        return o, S
    do = torch.zeros(T, E, H, Dv, dtype=torch.float64) if do is None else do.double()
    X = torch.zeros(E, H, Dk, Dv, dtype=torch.float64) if dlast is None else dlast.double().clone()
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for t in reversed(range(T)):
        X = X + scale * torch.einsum("ehi,ehj->ehij", q[t], do[t])
        dq[t] = scale * torch.einsum("ehij,ehj->ehi", states[t], do[t])
        dk[t] = torch.einsum("ehij,ehj->ehi", X, v[t])
        dv[t] = torch.einsum("ehij,ehi->ehj", X, k[t])
        X = torch.where(cut[t][:, None, None, None], torch.zeros_like(X), X * decay[None, :, None, None])
    return o, S, dq, dk, dv, X


def kept(y, group=128):
    """Codes and scales of the rows of y (already in its stored type), with the
    float32 arithmetic that defines them, one group at a time."""
    y = y.float()
    rows, n = y.shape
    codes, scales = torch.zeros(rows, n, dtype=torch.int8), torch.zeros(rows, -(-n // group))
    for r in range(rows):
        for g in range(scales.shape[1]):
            part = y[r, g * group:(g + 1) * group]
            scale = part.abs().max() * torch.tensor(1.0 / 127.0, dtype=torch.float32)
            if scale < torch.finfo(torch.float32).tiny:
                continue
            scales[r, g] = scale
            if torch.isfinite(scale):
                codes[r, g * group:(g + 1) * group] = torch.round(part * (1.0 / scale)).to(torch.int8)
    return codes, scales


def error(got, want):
    """2-norm of the difference over that of the wanted values."""
    got, want = got.detach().cpu().double(), want.detach().cpu().double()
    assert got.shape == want.shape, (got.shape, want.shape)
    if want.numel() == 0:
        return 0.0
    norm = want.norm()
    off = (got - want).norm()
    return float(off / norm) if norm > 0 else float(off)


def bound(dtype, terms, roundings=1):
    """Allowed error.  bfloat16 has 8 significant bits: a rounding is at most
    2^-8 of the value, and independent ones (of the result, of operands of its
    products) add in the mean square.  float32: a sum of `terms` values is off
    by about sqrt(terms) roundings of 2^-24, taken four times, with eight more
    roundings around it."""
    if dtype == torch.bfloat16:
        return roundings ** 0.5 * 2.0 ** -8
    return 4 * (terms ** 0.5 + 8) * 2.0 ** -24
