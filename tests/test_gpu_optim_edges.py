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


@pytest.mark.parametrize("optimizer", ["adamw", "adamw8"])
def test_the_ppo_step_from_a_graph_is_the_eager_one_bit_for_bit(tmp_path, optimizer):
    """The same gradients: the same parameters, moments (codes and exponents), counts and learning rates."""
    from duck_gym_b200 import biped
    from duck_gym_b200.bam_env import BamEnv
    from duck_gym_b200.ppo import PPO, PPOConfig

    biped.write_bam(tmp_path, seed=0)
    env = BamEnv(tmp_path, num_envs=64, iterations=10, auto_reset=True, reward_enabled=True, seconds=0.1)
    agent = PPO(env, PPOConfig(steps_per_env=8, optimizer=optimizer, weight_decay=0.01, max_grad_norm=0.5), seed=0)
    for _ in range(2):   # moments are there, gradients lie in one buffer
        agent.rollout()
        agent.update()
    params = list(agent.policy.parameters())
    tensors = [*params, agent.optimizer.param_groups[0]["step"], agent._lr64, agent._lr]
    tensors += [t for p in params for t in agent.optimizer.state[p].values()]
    kinds = {t.dtype for t in tensors}
    assert kinds >= ({torch.int8, torch.uint8} if optimizer == "adamw8" else {torch.float32})
    saved = [t.detach().clone() for t in tensors]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        agent._step_apply()
    results = []
    for step in (graph.replay, agent._step_apply):
        with torch.no_grad():
            for t, v in zip(tensors, saved):
                t.copy_(v)
        g = torch.Generator("cuda")
        g.manual_seed(7)
        for k in range(4):
            agent._flat_grad.normal_(generator=g).mul_(0.01)
            agent._flat_grad[-1] = [0.05, 0.01, 0.001, 0.01][k]   # the schedule's distance: the rate falls, stays, rises
            step()
        results.append([t.detach().clone() for t in tensors])
    assert all(torch.equal(a, b) for a, b in zip(*results))
    assert not any(torch.equal(a, b) for a, b in zip(results[0][:len(params)], saved))


@pytest.mark.parametrize("optimizer", ["adam", "adamw", "adamw8"])
def test_ppo_with_a_parameter_that_nothing_uses(tmp_path, optimizer):
    """It has no gradient in the first update, and one of zero in the captured ones."""
    from duck_gym_b200 import biped
    from duck_gym_b200.bam_env import BamEnv
    from duck_gym_b200.ppo import PPO, PPOConfig

    class Idle(PPO):
        def _make_policy(self, env):
            policy = super()._make_policy(env)
            policy.idle = torch.nn.Parameter(torch.ones(5))
            return policy

    biped.write_bam(tmp_path, seed=0)
    env = BamEnv(tmp_path, num_envs=64, iterations=10, auto_reset=True, reward_enabled=True, seconds=0.1)
    agent = Idle(env, PPOConfig(steps_per_env=8, optimizer=optimizer), seed=0)
    history = agent.learn(3)
    assert all(torch.isfinite(torch.tensor(list(h.values()))).all() for h in history)
    assert torch.equal(agent.policy.idle.detach(), torch.ones(5, device="cuda"))
    if optimizer != "adam":
        each = agent.cfg.epochs * agent.cfg.mini_batches
        assert int(agent.optimizer.param_groups[0]["step"]) == 3 * each
        assert int(agent.optimizer.state[agent.policy.idle]["step"]) == 2 * each
        assert not bool(agent.optimizer.state[agent.policy.idle]["exp_avg"].any())


def test_a_first_step_is_captured_after_prepare():
    params = [torch.nn.Parameter(torch.ones(300, device="cuda")) for _ in range(2)]
    opt = optim.AdamW(params, lr=1e-2, bits=8)
    params[0].grad = torch.full((300,), 0.5, device="cuda")
    opt.prepare()
    assert torch.equal(params[0].detach(), torch.ones(300, device="cuda")) and int(opt.param_groups[0]["step"]) == 0
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for _ in range(3):
        graph.replay()
    assert int(opt.param_groups[0]["step"]) == 3 and params[1] not in opt.state
    # Three steps of lr, whose gradient is always the same: codes of the moments are an eighth of an octave wide.
    assert bool(((params[0] - 0.97).abs() <= 0.03 * 0.13).all())


# (clipped, codes differ where the norms' last bits do)
@pytest.mark.parametrize("bits,clip", [(32, None), (32, 0.5), (8, None)])
def test_parameters_that_come_late_or_pause(bits, clip):
    """Several counts of steps in a group: the same as on the CPU, whose own test is against torch."""
    from test_optim_edges import PATTERN

    def run(device, steps=40):
        g = torch.Generator()
        g.manual_seed(4)
        params = [torch.nn.Parameter(torch.randn(700, generator=g).to(device)) for _ in PATTERN]
        opt = optim.AdamW([dict(params=params[:3]), dict(params=params[3:])], lr=1e-2, bits=bits, max_grad_norm=clip)
        for k in range(steps):
            for p, has in zip(params, PATTERN):
                grad = torch.randn(700, generator=g).to(device)
                p.grad = grad if has(k) else None
            opt.step()
        counts = [int(opt.state[p].get("step", opt.param_groups[0]["step"])) for p in params[:3]]
        return [p.detach().cpu() for p in params], [[t.cpu() for t in opt.state[p].values()] for p in params[:3]], counts

    (a, ms, counts), (b, ns, same) = run("cuda"), run("cpu")
    assert counts == same == [40, 30, 27]
    for x, y in zip(a, b):   # 40 steps of about lr, whose roots and quotients are off by 2^-20, and the parameter's own roundings
        assert bool(((x - y).abs() <= 40 * (1e-2 * 2.0 ** -18 + 2.0 ** -23 * (1 + y.abs()))).all())
    for x, y in zip(ms, ns):
        assert bits == 32 or all(torch.equal(s, t) for s, t in zip(x, y))
