"""CPU: calls of the gated operators (duck_gym_b200/memory.py) at the edges of what
their documentation allows."""

import pytest
import torch

from duck_gym_b200 import memory
from test_gated import layer


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_linear_gradients_inside_an_autocast_region(dtype):
    """The products of the backward pass are in float32 there, too."""
    case = layer(4, 20, 7, 11, dtype)
    leaves = [t.requires_grad_() for t in case[:5]]
    h = memory.gated_linear(*leaves)
    want = torch.autograd.grad(h, leaves, case[5], retain_graph=True)
    with torch.autocast("cpu", dtype=torch.bfloat16):
        got = torch.autograd.grad(h, leaves, case[5])
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_linear_derivatives_of_other_kinds_on_the_cpu():
    """Second derivatives, tangents and torch.func, as the plain operations have them."""
    x, wg, wu, bg, bu, _ = (t.double() for t in layer(5, 4, 3, 5))
    leaves = [t.requires_grad_() for t in (x, wg, wu, bg, bu)]
    call = lambda *t: memory.gated_linear(*t)
    assert torch.autograd.gradcheck(call, leaves, check_forward_ad=True)
    assert torch.autograd.gradgradcheck(call, leaves)
    want = torch.autograd.grad(call(*leaves).sum(), leaves)
    got = torch.func.grad(lambda *t: call(*t).sum(), argnums=(0, 1, 2, 3, 4))(*[t.detach() for t in leaves])
    assert all(torch.allclose(a, b) for a, b in zip(got, want))
    rows = torch.func.vmap(lambda row: call(row[None], wg, wu, bg, bu)[0])(x)
    assert torch.allclose(rows, call(x, wg, wu, bg, bu))
    # One argument alone, and no bias.
    _, tangent = torch.func.jvp(lambda w: call(x, wg, w), (wu.detach(),), (torch.ones_like(wu),))
    assert torch.allclose(tangent, torch.nn.functional.silu(x @ wg.t()) * x.sum(1, keepdim=True))
