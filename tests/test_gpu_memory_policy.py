"""GPU: the memory policy on the fused BAM environment, all operators together."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_steps_agree_with_the_rollout():
    from duck_gym_b200.memory_policy import MemoryActorCritic, MemoryPPOConfig

    torch.manual_seed(0)
    for bf16, tolerance in ((False, 1e-4), (True, 0.05)):
        # float32: sums in another order.  bfloat16: some ten roundings of 2^-8 on the way to outputs of order 1.
        policy = MemoryActorCritic(61, 76, 14, MemoryPPOConfig(bf16=bf16)).cuda()
        T, E = 24, 64
        obs, cobs = torch.randn(T, E, 61, device="cuda"), torch.randn(T, E, 76, device="cuda")
        resets = torch.rand(T, E, device="cuda") < 0.1
        state = torch.randn_like(policy.initial_state(E, "cuda"))
        with torch.no_grad():
            mu, value = policy.outputs(obs, cobs, state, resets)
            moving = state.clone()
            steps = [policy.outputs(obs[t], cobs[t], moving, resets[t]) for t in range(T)]
        for a, b in ((mu, torch.stack([s[0] for s in steps])), (value, torch.stack([s[1] for s in steps]))):
            assert a.dtype == torch.float32 and float((a - b).norm() / a.norm()) < tolerance


def test_gradients_agree_with_float64_on_the_cpu():
    from duck_gym_b200.memory_policy import MemoryActorCritic, MemoryPPOConfig

    torch.manual_seed(1)
    cfg = MemoryPPOConfig(bf16=False, width=64, heads=2, head_size=32, hidden=96)
    exact = MemoryActorCritic(9, 11, 3, cfg).double()
    T, E = 40, 6
    obs, cobs = torch.randn(T, E, 9, dtype=torch.float64), torch.randn(T, E, 11, dtype=torch.float64)
    resets, state = torch.rand(T, E) < 0.1, torch.randn(2, 1, E, 2, 32, 32, dtype=torch.float64)
    go, gv = torch.randn(T, E, 3, dtype=torch.float64), torch.randn(T, E, dtype=torch.float64)
    got = MemoryActorCritic(9, 11, 3, cfg).cuda()
    got.load_state_dict(exact.state_dict())
    results = []
    for policy, move in ((exact, lambda t: t), (got, lambda t: t.cuda().float() if t.is_floating_point() else t.cuda())):
        mu, value = policy.outputs(move(obs), move(cobs), move(state), move(resets))
        ((mu * move(go)).sum() + (value * move(gv)).sum()).backward()
        results.append({n: p.grad.cpu().double() for n, p in policy.named_parameters() if n != "std"})
    for name, want in results[0].items():
        # The outputs of the trunk are float32 in both; an 8-bit code on the edge between two may fall the other way.
        assert float((results[1][name] - want).norm() / want.norm()) < 2e-3, name


def test_memory_ppo_on_bam_env(tmp_path):
    from duck_gym_b200 import biped
    from duck_gym_b200.bam_env import BamEnv
    from duck_gym_b200.memory_policy import MemoryPPO, MemoryPPOConfig

    biped.write_bam(tmp_path, seed=0)
    env = BamEnv(tmp_path, num_envs=256, iterations=10, auto_reset=True, reward_enabled=True, seconds=0.1)
    agent = MemoryPPO(env, MemoryPPOConfig(steps_per_env=8), seed=0)
    before = torch.cat([p.detach().flatten() for p in agent.policy.parameters()]).clone()
    history = agent.learn(3)
    after = torch.cat([p.detach().flatten() for p in agent.policy.parameters()])
    assert torch.isfinite(after).all() and not torch.equal(before, after)
    assert all(torch.isfinite(torch.tensor(list(h.values()))).all() for h in history)
    s = agent.storage
    assert s.dones.sum() > 0 and torch.equal(agent.resets[1:], s.dones[:-1] != 0)
    assert torch.isfinite(agent.state).all() and agent.state.abs().sum() > 0
    # The captured step moves the states as the plain one does.
    state, obs, cobs = agent.state.clone(), agent.obs.clone(), agent.critic_obs.clone()
    with torch.no_grad():
        _, _, mu, _, value = [t.clone() for t in agent._act_graphed(obs, cobs)]
        moved = agent.state.clone()
        agent.state.copy_(state)
        _, _, mu2, _, value2 = agent._act(obs, cobs)
    assert torch.equal(mu, mu2) and torch.equal(value, value2) and torch.equal(moved, agent.state)
