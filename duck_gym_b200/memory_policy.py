"""A policy with memory for the PPO of ``ppo.py``, on the operators of
``memory.py``.

The reference trains a feed-forward actor-critic (scripts/train_bam_native.py:
14-140); rsl-rl's recurrent variant has an LSTM in front of the same MLPs.  Here
actor and critic each are

    h = Linear(obs)
    per block:  h = h + Linear(norm(attention(norm(h))))     memory
                h = h + MLP(norm(h))                         hidden layer in 8 bits
    out = Linear(norm(h))

with layer norms, linear attention with one decay per head (memories of 4 to 256
steps; its state is the memory of an environment) and an ELU layer whose output is
kept in 8 bits for the backward pass.  A rollout advances the states by single
steps; the update runs whole rollouts, from the states that they began with, with
episode ends inside them (gradients stay within a rollout, as rsl-rl's do).

    python -m duck_gym_b200.memory_policy [--envs N] [--iterations N]

trains one on the synthetic biped's velocity task.
"""

from __future__ import annotations

import warnings
from dataclasses import dataclass

import torch
from torch import nn

from . import memory
from .ppo import PPO, PPOConfig, ppo_loss


@dataclass
class MemoryPPOConfig(PPOConfig):
    learning_rate: float = 1e-4
    width: int = 256         # of the residual stream
    blocks: int = 1
    heads: int = 4
    head_size: int = 64      # of queries, keys and values
    hidden: int = 512        # of a block's MLP
    shortest: float = 4.0    # steps that the fastest and the slowest head remember
    longest: float = 256.0
    graph_update: bool = False   # minibatches run eagerly, whatever is set here


class LayerNorm(nn.Module):
    def __init__(self, width):
        super().__init__()
        self.weight, self.bias = nn.Parameter(torch.ones(width)), nn.Parameter(torch.zeros(width))

    def forward(self, x):
        return memory.layer_norm(x, self.weight, self.bias)


class MemoryBlock(nn.Module):
    def __init__(self, cfg: MemoryPPOConfig):
        super().__init__()
        inner = cfg.heads * cfg.head_size
        self.shape = (3, cfg.heads, cfg.head_size)
        self.norm, self.qkv, self.out = LayerNorm(cfg.width), nn.Linear(cfg.width, 3 * inner), nn.Linear(inner, cfg.width)
        self.mlp_norm = LayerNorm(cfg.width)
        self.up, self.down = nn.Linear(cfg.width, cfg.hidden), nn.Linear(cfg.hidden, cfg.width)
        # An evenly spaced ladder of memories, in their logarithm: decay = 1 - 1 / steps.
        steps = torch.logspace(0, 1, cfg.heads, base=cfg.longest / cfg.shortest) * cfg.shortest
        self.register_buffer("decay", 1.0 - 1.0 / steps)

    def forward(self, x, state, resets):
        """x [T, E, width] or, for one step without gradients, [E, width] with
        the state advanced in place."""
        qkv = self.qkv(self.norm(x)).unflatten(-1, self.shape)
        q, k, v = qkv.unbind(-3)
        if x.dim() == 2:
            o = memory.linear_attention_step(q, k, v, self.decay, state, resets)
        else:
            o, _ = memory.linear_attention(q, k, v, self.decay, state, resets, final_state=False)
        # The size of a sum over steps says little: each head's output is normed by itself.
        x = x + self.out(memory.layer_norm(o).flatten(-2))
        h = self.mlp_norm(x)
        rows = h.reshape(-1, h.shape[-1])
        y = memory.checkpointed_mlp(rows.to(qkv.dtype), *zip(*[(w.to(qkv.dtype), b.to(qkv.dtype)) for w, b in (
            (self.up.weight, self.up.bias), (self.down.weight, self.down.bias))]))
        return x + y.view(x.shape)


class MemoryTrunk(nn.Module):
    def __init__(self, inputs, outputs, cfg: MemoryPPOConfig):
        super().__init__()
        self.bf16 = cfg.bf16
        self.inner = nn.Linear(inputs, cfg.width)
        self.blocks = nn.ModuleList(MemoryBlock(cfg) for _ in range(cfg.blocks))
        self.norm, self.head = LayerNorm(cfg.width), nn.Linear(cfg.width, outputs)

    def forward(self, obs, states, resets):
        with torch.autocast(obs.device.type, dtype=torch.bfloat16, enabled=self.bf16, cache_enabled=False):
            x = self.inner(obs)
            for block, state in zip(self.blocks, states):
                x = block(x, state, resets)
            return self.head(self.norm(x)).float()


class MemoryActorCritic(nn.Module):
    """States are [2, blocks, E, heads, size, size] float32: the actor's and the
    critic's."""

    def __init__(self, actor_obs, critic_obs, actions, cfg: MemoryPPOConfig):
        super().__init__()
        self.cfg = cfg
        self.actor, self.critic = MemoryTrunk(actor_obs, actions, cfg), MemoryTrunk(critic_obs, 1, cfg)
        self.std = nn.Parameter(torch.full((actions,), float(cfg.initial_std)))

    def initial_state(self, envs, device=None):
        c = self.cfg
        return torch.zeros(2, c.blocks, envs, c.heads, c.head_size, c.head_size, device=device)

    def outputs(self, obs, critic_obs, states, resets):
        """Means and values of one step ([E, ...], states advanced in place) or
        of a rollout ([T, E, ...])."""
        return self.actor(obs, states[0], resets), self.critic(critic_obs, states[1], resets).squeeze(-1)


class _Computed:
    """Outputs of a policy in the place of the policy, for ppo_loss."""

    def __init__(self, mu, std, value):
        self.mu, self.std, self.v = mu, std, value

    def mean(self, obs):
        return self.mu

    def value(self, obs):
        return self.v

    def distribution(self, obs):
        return torch.distributions.Normal(self.mu, self.std.expand_as(self.mu), validate_args=False)


class MemoryPPO(PPO):
    """PPO whose minibatches are environments, with all of their steps.  Rollout
    steps replay a CUDA graph (``graph_rollout``), updates run eagerly."""

    def __init__(self, env, cfg: MemoryPPOConfig | None = None, device=None, seed=0):
        super().__init__(env, cfg or MemoryPPOConfig(), device, seed)
        if self.cfg.graph_update:
            warnings.warn("MemoryPPO's updates run eagerly: graph_update is not used")
        E = env.num_envs
        if E < self.cfg.mini_batches:
            raise ValueError("fewer environments than minibatches")
        self.state = self.policy.initial_state(E, self.device)
        self.first_state = torch.zeros_like(self.state)      # before the rollout
        # An episode begins with this step: the first one of all, and those after an end.
        self.reset = torch.ones(E, dtype=torch.bool, device=self.device)
        self.resets = torch.zeros(self.cfg.steps_per_env, E, dtype=torch.bool, device=self.device)

    def _make_policy(self, env):
        return MemoryActorCritic(self.obs.shape[1], self.critic_obs.shape[1], env.num_actions, self.cfg)

    def _act(self, obs, critic_obs):
        mu, value = self.policy.outputs(obs, critic_obs, self.state, self.reset)
        d = torch.distributions.Normal(mu, self.policy.std.expand_as(mu), validate_args=False)
        actions = d.rsample()
        return actions, d.log_prob(actions).sum(-1), d.mean, d.stddev, value

    def _act_graphed(self, obs, critic_obs):
        if self._graph is not None:
            return super()._act_graphed(obs, critic_obs)
        kept = self.state.clone()
        super()._act_graphed(obs, critic_obs)   # warm-up, capture and a replay: the states moved on
        self.state.copy_(kept)
        self._graph.replay()
        return self._graph_out

    def _begin_rollout(self):
        self.first_state.copy_(self.state)

    def _before_step(self, t):
        self.resets[t].copy_(self.reset)

    def _after_step(self, done):
        self.reset.copy_(done != 0)

    def _last_values(self):
        return self.policy.critic(self.critic_obs, self.state[1].clone(), self.reset).squeeze(-1)

    def update(self, generator=None):
        s, cfg = self.storage, self.cfg
        self._updates += 1
        size = s.E // cfg.mini_batches
        data = (s.actions, s.log_prob, s.mu, s.sigma, s.values, s.returns, s.advantages)
        stats = []
        for _ in range(cfg.epochs):
            order = torch.randperm(s.E, device=self.device, generator=generator)
            for b in range(cfg.mini_batches):
                envs = order[b * size:(b + 1) * size]
                obs, critic_obs = s.obs[:, envs], s.critic_obs[:, envs]
                mu, value = self.policy.outputs(obs, critic_obs, self.first_state[:, :, envs], self.resets[:, envs])
                flat = lambda x: x.flatten(0, 1)
                loss, info = ppo_loss(_Computed(flat(mu), self.policy.std, flat(value)), flat(obs), flat(critic_obs),
                                      *[flat(x[:, envs]) for x in data], cfg)
                self._adapt(info["kl"])
                self.optimizer.zero_grad(set_to_none=False)
                loss.backward()
                self.reducer.finish()
                nn.utils.clip_grad_norm_(self.policy.parameters(), cfg.max_grad_norm)
                self._optimizer_step()
                stats.append(info)
        return {k: torch.stack([x[k] for x in stats]).mean().item() for k in stats[0]}


def main():
    import argparse
    import tempfile

    from . import biped
    from .bam_env import BamEnv

    parser = argparse.ArgumentParser(description="PPO with a memory policy on the synthetic biped's velocity task.")
    parser.add_argument("--envs", type=int, default=4096)
    parser.add_argument("--iterations", type=int, default=5)
    args = parser.parse_args()
    with tempfile.TemporaryDirectory() as model:
        biped.write_bam(model, seed=0)
        training = dict(command_ranges=[[-0.3, 0.3], [-0.3, 0.3], [-1.0, 1.0]], command_resample_seconds=1.0)
        env = BamEnv(model, num_envs=args.envs, iterations=10, auto_reset=True, reward_enabled=True, training=training)
        agent = MemoryPPO(env)
        for i in range(args.iterations):
            agent.rollout()
            stats = agent.update()
            print(i, f"reward {float(agent.storage.rewards.mean()):.4f}",
                  " ".join(f"{k} {v:.4f}" for k, v in stats.items()))


if __name__ == "__main__":
    main()
