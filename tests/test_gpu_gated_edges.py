"""GPU: calls of the gated operators (duck_gym_b200/memory.py) at the edges of what
their documentation allows."""

import pytest
import torch

from duck_gym_b200 import memory

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("activation", ["silu", "gelu", "sigmoid"])
@pytest.mark.parametrize("up", [0.125, -3e37])
def test_linear_activations_over_the_whole_range(activation, dtype, up):
    """What far negative projections leave is zero, however large the numbers beside it."""
    a = [3.0, 0.0, -1.5, -60.0, -87.0, -88.0, -95.0, -200.0, -1e4, -1e30, -1e36, -3e38] + ([200.0, 1e36, 3e38] if up > 0 else [])
    a = torch.tensor(a).to(dtype)
    F = a.numel()
    x, w = torch.zeros(1, 8, dtype=dtype), [torch.zeros(F, 8, dtype=dtype) for _ in range(2)]
    x[0, 0], w[0][:, 0], w[1][:, 0] = 1, a, up
    biases = [torch.zeros(F, dtype=dtype, device="cuda", requires_grad=True) for _ in range(2)]
    h = memory.gated_linear(x.cuda(), w[0].cuda(), w[1].cuda(), *biases, activation=activation)
    got = (h[0], *torch.autograd.grad(h, biases, torch.full((1, F), 0.25, dtype=dtype, device="cuda")))
    A, u = a.double(), w[1][:, 0].double()
    s, rest = 1 / (1 + torch.exp(-A)), 1 / (1 + torch.exp(A))
    if activation == "gelu":
        s = torch.special.ndtr(A)
        y, slope = A * s, s + A * torch.exp(-A * A / 2) / (2 * torch.pi) ** 0.5
        # 1 + erf cancels: off by 2^-23 of 1, where it is not 0.
        lost = torch.where((A < 0) & (A > -20), 2.0 ** -23 * A.abs(), 0.0)
    else:
        y, slope = (A * s, s + A * s * rest) if activation == "silu" else (s, s * rest)
        # 1 / (1 + exp) may be flushed below the smallest normal number, 2^-126; times 100 at most.
        lost = torch.where(A > -100, 2.0 ** -119, 0.0)
    # Hardware's exponentials and quotients, with arguments of up to 128: 2^-18; the result's rounding; and denormals.
    relative = 2.0 ** -18 + (2.0 ** -8 if dtype == torch.bfloat16 else 0)
    for value, want, factor in zip(got, (y * u, 0.25 * u * slope, 0.25 * y), (u, u, torch.ones_like(u))):
        off = (value.detach().cpu().double() - want).abs()
        assert bool((off <= relative * want.abs() + lost * factor.abs() + 2.0 ** -124).all()), (off, want)
