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
