"""CPU: the memory policy with a gated recurrence and a gated linear layer
(duck_gym_b200/memory_policy.py), and PPO with the optimizer of optim.py."""

import pytest
import torch

from duck_gym_b200.memory_policy import MemoryActorCritic, MemoryPPO, MemoryPPOConfig
from duck_gym_b200.ppo import PPO, PPOConfig
from test_memory_policy import RecallEnv

SMALL = dict(bf16=False, width=16, heads=2, head_size=8, hidden=24, blocks=2)
KINDS = [dict(memory="recurrence"), dict(mlp="gated"), dict(memory="recurrence", mlp="gated")]


@pytest.mark.parametrize("kind", KINDS)
def test_steps_agree_with_the_rollout(kind):
    torch.manual_seed(0)
    policy = MemoryActorCritic(5, 7, 3, MemoryPPOConfig(**SMALL, **kind))
    T, E = 9, 4
    obs, cobs = torch.randn(T, E, 5), torch.randn(T, E, 7)
    resets = torch.rand(T, E) < 0.3
    state = torch.randn_like(policy.initial_state(E))
    with torch.no_grad():
        mu, value = policy.outputs(obs, cobs, state, resets)
        moving = state.clone()
        for t in range(T):
            m, v = policy.outputs(obs[t], cobs[t], moving, resets[t])
            assert torch.allclose(m, mu[t], atol=1e-5) and torch.allclose(v, value[t], atol=1e-5)


@pytest.mark.parametrize("kind", KINDS)
def test_every_parameter_gets_a_gradient_as_differences_say(kind):
    torch.manual_seed(0)
    policy = MemoryActorCritic(5, 7, 3, MemoryPPOConfig(**{**SMALL, "blocks": 1}, **kind)).double()
    obs, cobs = torch.randn(6, 4, 5).double(), torch.randn(6, 4, 7).double()
    state, resets = torch.randn_like(policy.initial_state(4)).double(), torch.rand(6, 4) < 0.2
    loss = lambda: sum((y.square() * (1 + i)).sum() for i, y in enumerate(policy.outputs(obs, cobs, state, resets)))
    loss().backward()
    for name, p in policy.named_parameters():
        assert name == "std" or (p.grad is not None and bool(p.grad.abs().sum() > 0)), name
        # Along the gradient, by central differences: the loss is smooth but for the 8-bit codes of the ELU layer.  The
        # trunk's outputs are float32, so that a loss of some 50 is known to 2 * 50 * 2^-24 = 6e-6 at best, two of them.
        # (Through the attention's norm of each head the differences' own error, which goes with h^2, is 3e-3 at this h.)
        if name == "std" or kind != KINDS[2]:
            continue
        h = 1e-3 / float(p.grad.norm())
        with torch.no_grad():
            p += h * p.grad
            up = float(loss())
            p -= 2 * h * p.grad
            down = float(loss())
            p += h * p.grad
        expected = 2 * h * float(p.grad.square().sum())
        assert abs(up - down - expected) <= 1e-3 * expected + 1.2e-5, name


def test_ladder_of_gates():
    torch.manual_seed(0)
    block = MemoryActorCritic(5, 7, 3, MemoryPPOConfig(**SMALL, memory="recurrence")).actor.blocks[0]
    kept = torch.sigmoid(block.gate_value.bias[:16])
    assert torch.allclose(1 / (1 - kept[[0, -1]]), torch.tensor([4.0, 256.0]), rtol=1e-3)


@pytest.mark.parametrize("optimizer", ["adamw", "adamw8"])
def test_memory_ppo_runs(optimizer):
    agent = MemoryPPO(RecallEnv(n=16), MemoryPPOConfig(**SMALL, memory="recurrence", mlp="gated", steps_per_env=6,
                                                       optimizer=optimizer, weight_decay=0.01), device="cpu")
    before = [p.detach().clone() for p in agent.policy.parameters()]
    for stats in agent.learn(2):
        assert all(x == x for x in stats.values())
    assert all(not torch.equal(a, b) and bool(b.isfinite().all()) for a, b in zip(before, agent.policy.parameters()))
    group, = agent.optimizer.param_groups
    assert int(group["step"]) == 2 * agent.cfg.epochs * agent.cfg.mini_batches


def test_one_step_agrees_with_adam():
    """Without weight decay it is Adam; one minibatch, so that differences do not grow."""
    results = []
    for optimizer in ("adam", "adamw"):
        cfg = PPOConfig(bf16=False, steps_per_env=6, epochs=1, mini_batches=1, actor_hidden=(16,), critic_hidden=(16,),
                        optimizer=optimizer, max_grad_norm=0.1)
        agent = PPO(RecallEnv(n=16), cfg, device="cpu")
        agent.rollout()
        agent.update(torch.Generator().manual_seed(0))
        results.append([p.detach().clone() for p in agent.policy.parameters()])
    for a, b in zip(*results):
        assert float((a - b).abs().max()) <= 1e-5 * 3e-4 + 2.0 ** -22 * float(a.abs().max()) + 1e-8


def test_refusals():
    for wrong in (dict(memory="lstm"), dict(mlp="relu")):
        with pytest.raises(ValueError):
            MemoryPPOConfig(**wrong)
    with pytest.raises(ValueError):
        PPO(RecallEnv(n=4), PPOConfig(optimizer="sgd"), device="cpu")
