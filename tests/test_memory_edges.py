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
