"""GPU: calls of the optimizer (duck_gym_b200/optim.py) at the edges of what its
documentation allows."""

import pytest
import torch

from duck_gym_b200 import optim

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
def test_a_first_step_is_not_captured(bits):
    """Its moments would be zeroed by every replay."""
    params = [torch.nn.Parameter(torch.ones(300, device="cuda")) for _ in range(2)]
    opt = optim.AdamW(params, lr=1e-2, bits=bits)
    for p in params:
        p.grad = torch.full((300,), 0.5, device="cuda")
    with pytest.raises(RuntimeError, match="captured"), torch.cuda.graph(torch.cuda.CUDAGraph()):
        opt.step()
    torch.cuda.synchronize()
    assert all(torch.equal(p.detach(), torch.ones(300, device="cuda")) for p in params)
    opt.step()
    params[1].grad = None   # its own count would be made by every replay, too
    with pytest.raises(RuntimeError, match="captured"), torch.cuda.graph(torch.cuda.CUDAGraph()):
        opt.step()
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for _ in range(3):
        graph.replay()
    assert int(opt.param_groups[0]["step"]) == 5 and int(opt.state[params[1]]["step"]) == 1
    # The other one's five steps of lr, as a run without graphs has them.
    p = torch.nn.Parameter(torch.ones(300, device="cuda"))
    plain = optim.AdamW([p], lr=1e-2, bits=bits)
    p.grad = torch.full((300,), 0.5, device="cuda")
    for _ in range(5):
        plain.step()
    assert torch.equal(p, params[0])
