"""CPU: calls of the optimizer (duck_gym_b200/optim.py) at the edges of what its
documentation allows."""

import pytest
import torch

from duck_gym_b200 import optim


def count():
    return torch.zeros((), dtype=torch.int64)


@pytest.mark.parametrize("bits", [32, 8])
def test_iterators_are_taken_as_lists_are(bits):
    def tensors():
        p, g = [torch.ones(5), torch.ones(3)], [torch.full((5,), 0.5), torch.full((3,), -2.0)]
        if bits == 8:
            return p, g, [optim.state8_zeros(x, True) for x in p], [optim.state8_zeros(x, False) for x in p]
        return p, g, [torch.zeros_like(x) for x in p], [torch.zeros_like(x) for x in p]

    lists, iterators, a, b = tensors(), tensors(), count(), count()
    optim.adamw_step(*lists, a, 0.1, max_norm=1.0)
    optim.adamw_step(*map(iter, iterators), b, 0.1, max_norm=1.0)
    assert int(a) == int(b) == 1 and not torch.equal(lists[0][0], torch.ones(5))
    flat = lambda x: [t for s in x for t in (flat(s) if isinstance(s, (list, tuple)) else [s])]
    assert all(torch.equal(x, y) for x, y in zip(flat(lists), flat(iterators)))


@pytest.mark.parametrize("lr", [float("nan"), float("inf"), -float("inf")])
def test_a_learning_rate_that_is_not_finite_is_refused(lr):
    p, step = torch.ones(4), count()
    with pytest.raises(RuntimeError, match="finite"):
        optim.adamw_step([p], [torch.ones(4)], [torch.zeros(4)], [torch.zeros(4)], step, lr)
    assert torch.equal(p, torch.ones(4)) and int(step) == 0
