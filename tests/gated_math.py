"""Plain float64 restatements of the gated operators and of the optimizer for
their tests, on the CPU, written from the formulas."""

import torch


def recurrence(gates, values, state, resets, dout=None, dlast=None):
    """(out, last) and, with dout or dlast, (out, last, dgates, dvalues, dstate)."""
    T, E, N = gates.shape
    f, c = 1 / (1 + torch.exp(-gates.double())), values.double()
    rest = 1 / (1 + torch.exp(gates.double()))
    h = torch.zeros(E, N, dtype=torch.float64) if state is None else state.double().clone()
    cut = torch.zeros(T, E, dtype=torch.bool) if resets is None else resets.bool()
    out, before = torch.zeros(T, E, N, dtype=torch.float64), []
    for t in range(T):
        h = torch.where(cut[t][:, None], torch.zeros_like(h), h)
        before.append(h)
        h = f[t] * h + rest[t] * c[t]
        out[t] = h
    if dout is None and dlast is None:
        return out, h
    dout = torch.zeros(T, E, N, dtype=torch.float64) if dout is None else dout.double()
    x = torch.zeros(E, N, dtype=torch.float64) if dlast is None else dlast.double().clone()
    dg, dc = torch.zeros_like(c), torch.zeros_like(c)
    for t in reversed(range(T)):
        dh = x + dout[t]
        dc[t] = dh * rest[t]
        dg[t] = dh * (before[t] - c[t]) * f[t] * rest[t]
        x = torch.where(cut[t][:, None], torch.zeros_like(x), dh * f[t])
    return out, h, dg, dc, x


def adamw(p, g, m, v, t, lr, betas, eps, weight_decay, clip=1.0):
    """New (p, m, v) of one tensor after step number t."""
    p, g, m, v = (x.double() for x in (p, g, m, v))
    g = g * clip
    m, v = betas[0] * m + (1 - betas[0]) * g, betas[1] * v + (1 - betas[1]) * g * g
    step = m / (1 - betas[0] ** t) / ((v / (1 - betas[1] ** t)).sqrt() + eps)
    return p - lr * weight_decay * p - lr * step, m, v


def hashed(t, place, n):
    """The random bits of the first n values of the place-th tensor at step t."""
    def mix(x):
        x = (x ^ x >> 16) * 0x85EBCA6B % 2**32
        x = (x ^ x >> 13) * 0xC2B2AE35 % 2**32
        return x ^ x >> 16
    key = mix((t + 0x9E3779B9 * (place + 1)) % 2**32)
    return [mix(key ^ i) for i in range(n)]


def code_values(codes, exponents):
    """What a moment in 8 bits stands for, value by value: an octave and eighths."""
    most, flat = 127 if codes.dtype == torch.int8 else 255, codes.reshape(-1).tolist()
    out = []
    for i, c in enumerate(flat):
        e = int(exponents[i // 128])
        octave, eighths = divmod(abs(c) + max(0, 8 * e + 8 - most), 8)
        value = 2.0 ** (octave - 127) * (1 + eighths / 8) if octave else eighths * 2.0 ** -129
        out.append(float("nan") if e == 255 else 0.0 if c == 0 else value if c > 0 else -value)
    return torch.tensor(out, dtype=torch.float64).view(codes.shape)


def linear(x, w_gate, w_up, b_gate, b_up, activation, dh=None):
    """h and, with dh, (h, dx, dw_gate, dw_up, db_gate, db_up) for rows x."""
    x, w_gate, w_up = x.double(), w_gate.double(), w_up.double()
    a = x @ w_gate.t() + (0.0 if b_gate is None else b_gate.double())
    u = x @ w_up.t() + (0.0 if b_up is None else b_up.double())
    s = torch.special.ndtr(a) if activation == "gelu" else 1 / (1 + torch.exp(-a))
    ds = torch.exp(-a * a / 2) / (2 * torch.pi) ** 0.5 if activation == "gelu" else s * (1 - s)
    y, slope = (s, ds) if activation == "sigmoid" else (a * s, s + a * ds)
    if dh is None:
        return y * u
    da, du = dh.double() * u * slope, dh.double() * y
    return y * u, da @ w_gate + du @ w_up, da.t() @ x, du.t() @ x, da.sum(0), du.sum(0)
