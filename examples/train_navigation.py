"""Trains a policy on the navigation scenario: rollouts of ``Environment.step``, ``gae``, the clipped
policy loss and ``AdamW``, all on the HIP device.

    python examples/train_navigation.py --head gaussian
    python examples/train_navigation.py --head categorical --bits 8
    python examples/train_navigation.py --head categorical --memory 4 --clone 10

The Gaussian head acts in the two continuous velocity commands; the categorical one chooses among
nine of them (eight directions and standing still).  ``--memory`` gives the policy that many heads of
``decay_attention`` along the episode, ``decay_attention_step`` while it acts.  ``--clone`` begins
with iterations of imitation: the policy acts and learns, by ``linear_cross_entropy``, which of the
nine moves points to the agent's goal.
"""

from __future__ import annotations

import argparse
import math
import os
import sys

import torch
from torch import nn

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))

from swarp_amd import (AdamW, Environment, NavigationScenario, categorical_policy_loss,  # noqa: E402
                       decay_attention, decay_attention_step, gae, gaussian_policy_loss,
                       linear_cross_entropy)


class Memory(nn.Module):
    """What the steps of an episode leave behind: heads of linear attention, each with a decay."""

    def __init__(self, width: int, heads: int) -> None:
        super().__init__()
        self.heads = heads
        self.qkv = nn.Linear(width, 3 * width)
        self.mix = nn.Linear(width, width)
        # half of what was seen is forgotten after 2, 4, 8.. steps
        self.register_buffer("log_decay", -math.log(2.0) * 0.5 ** torch.arange(1.0, heads + 1))

    def empty(self, *batch: int) -> torch.Tensor:
        n = self.mix.in_features // self.heads
        return torch.zeros(*batch, self.heads, n, n, device=self.log_decay.device)

    def _heads(self, h: torch.Tensor):
        return self.qkv(h).unflatten(-1, (3, self.heads, -1)).unbind(-3)

    def forward(self, h: torch.Tensor, state: torch.Tensor, starts: torch.Tensor) -> torch.Tensor:
        return h + self.mix(decay_attention(*self._heads(h), self.log_decay, state,
                                            starts).out.flatten(-2))

    def step(self, h: torch.Tensor, state: torch.Tensor, starts: torch.Tensor) -> torch.Tensor:
        return h + self.mix(decay_attention_step(*self._heads(h), self.log_decay, state,
                                                 starts).flatten(-2))


class Policy(nn.Module):
    """Two-layer trunk, with or without a memory, an action head and a value head, shared by all
    agents."""

    def __init__(self, obs_dim: int, act_dim: int, head: str, width: int = 64,
                 memory: int = 0) -> None:
        super().__init__()
        self.head = head
        self.trunk = nn.Sequential(nn.Linear(obs_dim, width), nn.Tanh(), nn.Linear(width, width),
                                   nn.Tanh())
        self.out = nn.Linear(width, 9 if head == "categorical" else act_dim)
        self.value = nn.Linear(width, 1)
        self.memory = Memory(width, memory) if memory else None
        self.log_std = nn.Parameter(torch.full((act_dim,), -0.5)) if head == "gaussian" else None
        # unit commands of the nine choices
        turn = torch.arange(8) * (math.pi / 4)
        moves = torch.cat([torch.stack([turn.cos(), turn.sin()], -1), torch.zeros(1, 2)])
        self.register_buffer("moves", moves)
        with torch.no_grad():
            self.out.weight.mul_(0.01)

    def features(self, obs: torch.Tensor, state=None, starts=None) -> torch.Tensor:
        """Of a rollout's steps, which come first where there is a memory."""
        h = self.trunk(obs)
        return h if self.memory is None else self.memory(h, state, starts)

    def forward(self, obs: torch.Tensor, state=None, starts=None):
        h = self.features(obs, state, starts)
        return self.out(h), self.value(h).squeeze(-1)

    def step(self, obs: torch.Tensor, state=None, starts=None):
        """One step of :meth:`forward`, with ``state`` brought forward."""
        h = self.trunk(obs)
        if self.memory is not None:
            h = self.memory.step(h, state, starts)
        return self.out(h), self.value(h).squeeze(-1)

    @torch.no_grad()
    def value_after(self, obs: torch.Tensor, state=None, starts=None) -> torch.Tensor:
        """Value of what comes next, which is not acted on: ``state`` stays."""
        return self.step(obs, None if state is None else state.clone(), starts)[1]

    @torch.no_grad()
    def act(self, obs: torch.Tensor, state=None, starts=None):
        """(what the policy chose, the environment's actions, the log-probability, the value)."""
        out, value = self.step(obs, state, starts)
        if self.head == "categorical":
            logp = torch.log_softmax(out, -1)
            choice = torch.argmax(logp - torch.log(-torch.log(torch.rand_like(logp))), -1)
            return choice, self.moves[choice], logp.gather(-1, choice[..., None])[..., 0], value
        std = self.log_std.exp()
        choice = out + std * torch.randn_like(out)
        z = (choice - out) / std
        logp = (-0.5 * z * z - self.log_std - 0.5 * math.log(2 * math.pi)).sum(-1)
        return choice, choice, logp, value


def expert(policy: Policy, obs: torch.Tensor) -> torch.Tensor:
    """The move that points to the goal; standing still close to it."""
    to = obs[..., 7:9]  # (the goal's place, seen from the agent)
    best = (to @ policy.moves[:8].t()).argmax(-1)
    return torch.where(to.norm(dim=-1) < 0.05, 8, best)


def train(head: str = "gaussian", bits: int = 32, n_envs: int = 1024, n_agents: int = 4,
          steps: int = 32, iterations: int = 50, epochs: int = 4, lr: float = 3e-3, seed: int = 0,
          device: str = "cuda:0", log=print, memory: int = 0, clone: int = 0) -> list[float]:
    """Mean reward per step of every iteration."""
    if clone and head != "categorical":
        raise ValueError("only the categorical head's moves are imitated")
    torch.manual_seed(seed)
    env = Environment(NavigationScenario(n_agents=n_agents, world_size=1.0), n_envs=n_envs,
                      device=device, dt=0.1, max_steps=100, seed=seed, clone_outputs=True)
    policy = Policy(env.obs_dim, env.act_dim, head, 64, memory).to(device)
    opt = AdamW(policy.parameters(), lr=lr, bits=bits, max_grad_norm=0.5, seed=seed)
    obs = env.reset(seed=seed)
    state = policy.memory.empty(n_envs, n_agents) if memory else None
    starts = torch.ones(n_envs, dtype=torch.bool, device=device)
    going = torch.zeros_like(starts)
    history = []
    for it in range(clone + iterations):
        keep = {k: [] for k in ("obs", "choice", "logp", "value", "reward", "term", "trunc", "next",
                                "starts")}
        final, before = [], None if state is None else state.clone()
        for _ in range(steps):
            choice, action, logp, value = policy.act(*((obs, state, starts) if memory else (obs,)))
            new_obs, reward, terminated, truncated, _ = env.step(action)
            for k, v in zip(keep, (obs, choice, logp, value, reward, terminated, truncated,
                                   new_obs, starts)):
                keep[k].append(v)
            if memory and it >= clone:
                final.append(policy.value_after(new_obs, state, going))
            # (envs whose episode ended begin another; what they ended in is kept above)
            starts = terminated | truncated
            obs = env.reset_at(starts).clone()
        roll = {k: torch.stack(v) for k, v in keep.items()}
        seen = (roll["obs"], before, roll["starts"]) if memory else (roll["obs"],)
        history.append(float(roll["reward"].mean()))
        if it < clone:
            moves = expert(policy, roll["obs"])
            for _ in range(epochs):
                opt.zero_grad(set_to_none=True)
                same = linear_cross_entropy(policy.features(*seen), policy.out.weight, moves,
                                            policy.out.bias)
                same.loss.backward()
                opt.step()
            log(f"imitation {it}: reward {history[-1]:.4f}  loss {float(same.loss.detach()):.4f}")
            continue
        with torch.no_grad():
            last = policy.value_after(obs, state, starts) if memory else policy(obs)[1]
            # at a time limit the return goes on with the value of what the episode ended in
            adv, returns = gae(roll["reward"], torch.cat([roll["value"], last[None]]), roll["term"],
                               roll["trunc"],
                               torch.stack(final) if memory else policy(roll["next"])[1],
                               gamma=0.99, lam=0.95)
            adv = (adv - adv.mean()) / (adv.std() + 1e-6)
        for _ in range(epochs):
            opt.zero_grad(set_to_none=True)
            out, value = policy(*seen)
            if head == "categorical":
                pg = categorical_policy_loss(out, roll["choice"], roll["logp"], adv,
                                             entropy_coef=0.005)
            else:
                pg = gaussian_policy_loss(out, policy.log_std, roll["choice"], roll["logp"], adv,
                                          entropy_coef=0.001)
            (pg.loss + 0.5 * (value - returns).square().mean()).backward()
            opt.step()
        if (it - clone) % 10 == 0 or it == clone + iterations - 1:
            log(f"iteration {it - clone}: reward {history[-1]:.4f}  entropy {float(pg.entropy):.3f}  "
                f"kl {float(pg.kl):.4f}  clipped {float(pg.clip_fraction):.3f}  "
                f"gradient norm {float(opt.last_grad_norm):.3f}")
    return history


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__,
                                 formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--head", choices=("gaussian", "categorical"), default="gaussian")
    ap.add_argument("--bits", type=int, choices=(8, 32), default=32)
    ap.add_argument("--envs", type=int, default=1024)
    ap.add_argument("--agents", type=int, default=4)
    ap.add_argument("--iterations", type=int, default=50)
    ap.add_argument("--memory", type=int, default=0, choices=(0, 1, 2, 4, 8),
                    help="heads of the policy's memory")
    ap.add_argument("--clone", type=int, default=0, help="iterations of imitation at first")
    ap.add_argument("--seed", type=int, default=0)
    a = ap.parse_args()
    train(a.head, a.bits, a.envs, a.agents, iterations=a.iterations, seed=a.seed,
          memory=a.memory, clone=a.clone)


if __name__ == "__main__":
    main()
