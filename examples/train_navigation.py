"""Trains a policy on the navigation scenario: rollouts of ``Environment.step``, ``gae``, the clipped
policy loss and ``AdamW``, all on the HIP device.

    python examples/train_navigation.py --head gaussian
    python examples/train_navigation.py --head categorical --bits 8

The Gaussian head acts in the two continuous velocity commands; the categorical one chooses among
nine of them (eight directions and standing still).
"""

from __future__ import annotations

import argparse
import math
import os
import sys

import torch
from torch import nn

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))

from swarp_amd import (AdamW, Environment, NavigationScenario, categorical_policy_loss, gae,  # noqa: E402
                       gaussian_policy_loss)


class Policy(nn.Module):
    """Two-layer trunk with an action head and a value head, shared by all agents."""

    def __init__(self, obs_dim: int, act_dim: int, head: str, width: int = 64) -> None:
        super().__init__()
        self.head = head
        self.trunk = nn.Sequential(nn.Linear(obs_dim, width), nn.Tanh(), nn.Linear(width, width),
                                   nn.Tanh())
        self.out = nn.Linear(width, 9 if head == "categorical" else act_dim)
        self.value = nn.Linear(width, 1)
        self.log_std = nn.Parameter(torch.full((act_dim,), -0.5)) if head == "gaussian" else None
        # unit commands of the nine choices
        turn = torch.arange(8) * (math.pi / 4)
        moves = torch.cat([torch.stack([turn.cos(), turn.sin()], -1), torch.zeros(1, 2)])
        self.register_buffer("moves", moves)
        with torch.no_grad():
            self.out.weight.mul_(0.01)

    def forward(self, obs: torch.Tensor):
        h = self.trunk(obs)
        return self.out(h), self.value(h).squeeze(-1)

    @torch.no_grad()
    def act(self, obs: torch.Tensor):
        """(what the policy chose, the environment's actions, the log-probability, the value)."""
        out, value = self(obs)
        if self.head == "categorical":
            logp = torch.log_softmax(out, -1)
            choice = torch.argmax(logp - torch.log(-torch.log(torch.rand_like(logp))), -1)
            return choice, self.moves[choice], logp.gather(-1, choice[..., None])[..., 0], value
        std = self.log_std.exp()
        choice = out + std * torch.randn_like(out)
        z = (choice - out) / std
        logp = (-0.5 * z * z - self.log_std - 0.5 * math.log(2 * math.pi)).sum(-1)
        return choice, choice, logp, value


def train(head: str = "gaussian", bits: int = 32, n_envs: int = 1024, n_agents: int = 4,
          steps: int = 32, iterations: int = 50, epochs: int = 4, lr: float = 3e-3, seed: int = 0,
          device: str = "cuda:0", log=print) -> list[float]:
    """Mean reward per step of every iteration."""
    torch.manual_seed(seed)
    env = Environment(NavigationScenario(n_agents=n_agents, world_size=1.0), n_envs=n_envs,
                      device=device, dt=0.1, max_steps=100, seed=seed, clone_outputs=True)
    policy = Policy(env.obs_dim, env.act_dim, head).to(device)
    opt = AdamW(policy.parameters(), lr=lr, bits=bits, max_grad_norm=0.5, seed=seed)
    obs = env.reset(seed=seed)
    history = []
    for it in range(iterations):
        keep = {k: [] for k in ("obs", "choice", "logp", "value", "reward", "term", "trunc", "next")}
        for _ in range(steps):
            choice, action, logp, value = policy.act(obs)
            new_obs, reward, terminated, truncated, _ = env.step(action)
            for k, v in zip(keep, (obs, choice, logp, value, reward, terminated, truncated,
                                   new_obs)):
                keep[k].append(v)
            # (envs whose episode ended begin another; what they ended in is kept above)
            obs = env.reset_at(terminated | truncated).clone()
        roll = {k: torch.stack(v) for k, v in keep.items()}
        with torch.no_grad():
            last = policy(obs)[1]
            # at a time limit the return goes on with the value of what the episode ended in
            adv, returns = gae(roll["reward"], torch.cat([roll["value"], last[None]]), roll["term"],
                               roll["trunc"], policy(roll["next"])[1], gamma=0.99, lam=0.95)
            adv = (adv - adv.mean()) / (adv.std() + 1e-6)
        for _ in range(epochs):
            opt.zero_grad(set_to_none=True)
            out, value = policy(roll["obs"])
            if head == "categorical":
                pg = categorical_policy_loss(out, roll["choice"], roll["logp"], adv,
                                             entropy_coef=0.005)
            else:
                pg = gaussian_policy_loss(out, policy.log_std, roll["choice"], roll["logp"], adv,
                                          entropy_coef=0.001)
            (pg.loss + 0.5 * (value - returns).square().mean()).backward()
            opt.step()
        history.append(float(roll["reward"].mean()))
        if it % 10 == 0 or it == iterations - 1:
            log(f"iteration {it}: reward {history[-1]:.4f}  entropy {float(pg.entropy):.3f}  "
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
    ap.add_argument("--seed", type=int, default=0)
    a = ap.parse_args()
    train(a.head, a.bits, a.envs, a.agents, iterations=a.iterations, seed=a.seed)


if __name__ == "__main__":
    main()
