"""CPU: the memory policy (duck_gym_b200/memory_policy.py): steps and rollouts
agree, states end with episodes, and it learns what a policy without memory
cannot."""

import torch

from duck_gym_b200.memory_policy import MemoryActorCritic, MemoryPPO, MemoryPPOConfig

SMALL = dict(bf16=False, width=16, heads=2, head_size=8, hidden=24, blocks=2)


def test_steps_agree_with_the_rollout():
    torch.manual_seed(0)
    policy = MemoryActorCritic(5, 7, 3, MemoryPPOConfig(**SMALL))
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
        # What came before an episode does not matter.
        other = obs.clone()
        last = [int(resets[:, e].nonzero().max()) if resets[:, e].any() else 0 for e in range(E)]
        for e in range(E):
            other[:last[e], e] += 1.0
        mu2, _ = policy.outputs(other, cobs, state, resets)
        for e in range(E):
            assert torch.equal(mu2[last[e]:, e], mu[last[e]:, e]) or not resets[:, e].any()
            if last[e]:
                assert not torch.equal(mu2[:last[e], e], mu[:last[e], e])


def test_every_parameter_gets_a_gradient():
    torch.manual_seed(0)
    policy = MemoryActorCritic(5, 7, 3, MemoryPPOConfig(**SMALL))
    mu, value = policy.outputs(torch.randn(6, 4, 5), torch.randn(6, 4, 7), policy.initial_state(4),
                               torch.zeros(6, 4, dtype=torch.bool))
    (mu.square().sum() + value.square().sum()).backward()
    for name, p in policy.named_parameters():
        assert name == "std" or (p.grad is not None and bool(p.grad.abs().sum() > 0)), name


class RecallEnv:
    """The target is shown at an episode's first step only; the reward is
    -|a - target|^2 at every step; episodes of 6 steps, ending at different times."""

    def __init__(self, n=64, seed=0):
        self.num_envs, self.num_actions, self.device = n, 1, torch.device("cpu")
        self.g = torch.Generator().manual_seed(seed)
        self.t = torch.arange(n) % 6
        self.target = self.draw(n)

    def draw(self, n):
        return (torch.rand(n, 1, generator=self.g) < 0.5).float() * 2 - 1

    def get_observations(self):
        first = (self.t == 0).float()[:, None]
        return torch.cat((self.target * first, first), -1)

    def step(self, actions):
        reward = -(actions - self.target).square().sum(-1)
        self.t = self.t + 1
        done = self.t >= 6
        self.t = torch.where(done, 0, self.t)
        self.target = torch.where(done[:, None], self.draw(self.num_envs), self.target)
        return self.get_observations(), reward, done, {"time_outs": torch.zeros_like(done)}


def test_learns_to_remember():
    agent = MemoryPPO(RecallEnv(), MemoryPPOConfig(bf16=False, width=32, heads=2, head_size=16, hidden=32, steps_per_env=24,
                                                   learning_rate=1e-3, initial_std=0.3, entropy_coef=0.0, gamma=0.5),
                      device="cpu")
    agent.learn(12)
    # Without memory the best is to answer 0: -1 - std^2 on five steps of six.
    assert float(agent.storage.rewards.mean()) > -0.6
    assert bool((agent.resets[1:] == (agent.storage.dones[:-1] != 0)).all())
