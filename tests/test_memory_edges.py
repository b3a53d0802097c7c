"""CPU: what the memory operators (duck_gym_b200/memory.py) have to refuse or
keep where autograd, autocast and states in place meet."""

import pytest
import torch

from duck_gym_b200 import memory


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def heads(g, *shape, count=3):
    return [torch.randn(*shape, generator=g) for _ in range(count)]


def test_step_refuses_a_state_that_requires_a_gradient():
    g = gen(0)
    q, k, v = heads(g, 3, 2, 4)
    decay = torch.tensor([0.7, 0.9])
    state = torch.randn(3, 2, 4, 4, generator=g, requires_grad=True)
    with pytest.raises(RuntimeError):
        memory.linear_attention_step(q, k, v, decay, state)
    with torch.no_grad():
        memory.linear_attention_step(q, k, v, decay, state)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_checkpointed_mlp_backward_inside_autocast(dtype):
    g = gen(1)
    sizes = (7, 40, 30, 3)
    w = [(torch.randn(o, i, generator=g) / i ** 0.5).to(dtype) for i, o in zip(sizes, sizes[1:])]
    b = [(0.1 * torch.randn(o, generator=g)).to(dtype) for o in sizes[1:]]
    leaves = [t.requires_grad_() for t in (torch.randn(50, 7, generator=g).to(dtype), *w, *b)]
    dy = torch.randn(50, 3, generator=g).to(dtype)
    run = lambda: memory.checkpointed_mlp(leaves[0], leaves[1:4], leaves[4:])
    want = torch.autograd.grad(run(), leaves, dy)
    y = run()
    with torch.autocast("cpu", dtype=torch.bfloat16):
        got = torch.autograd.grad(y, leaves, dy)
    assert all(torch.equal(a, c) for a, c in zip(got, want))   # the very products of the pass outside


def test_attention_backward_inside_autocast():
    g = gen(2)
    leaves = [t.requires_grad_() for t in (*heads(g, 9, 2, 2, 8), torch.randn(2, 2, 8, 8, generator=g))]
    decay, do = torch.tensor([0.5, 0.9]), torch.randn(9, 2, 2, 8, generator=g)
    run = lambda: memory.linear_attention(*leaves[:3], decay, leaves[3])[0]
    want = torch.autograd.grad(run(), leaves, do)
    out = run()
    with torch.autocast("cpu", dtype=torch.bfloat16):
        got = torch.autograd.grad(out, leaves, do)
    assert all(torch.equal(a, c) for a, c in zip(got, want))


def test_no_steps_give_a_state_of_its_own():
    S = torch.randn(2, 1, 4, 4, generator=gen(3))
    q = torch.zeros(0, 2, 1, 4)
    _, last = memory.linear_attention(q, q, q, torch.tensor([0.9]), S)
    assert torch.equal(last, S)
    last.zero_()   # as a control step would
    assert bool(S.abs().sum() > 0)
