"""What the training example hands to ``gae``: at a time limit, the value of the observation that
the episode ended in, not of the reset's nor of the one before."""

import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu


def example():
    path = Path(__file__).resolve().parents[1] / "examples" / "train_navigation.py"
    spec = importlib.util.spec_from_file_location("train_navigation", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_final_values_are_of_what_the_episode_ended_in(monkeypatch):
    mod = example()
    policies, ended, seen = [], [], []

    class Policy(mod.Policy):
        def __init__(self, *args):
            super().__init__(*args)
            policies.append(self)

    class Environment(mod.Environment):
        def step(self, actions):
            out = super().step(actions)
            ended.append(out[0].clone())
            return out

    def gae(rewards, values, terminated, truncated, final_values, **kw):
        obs = torch.stack(ended)
        ended.clear()
        with torch.no_grad():
            want = policies[0](obs)[1]
        at = truncated & ~terminated
        assert torch.allclose(final_values[at], want[at], rtol=1e-5, atol=1e-6)
        # the next step's observation is the reset's
        if bool(at[:-1].any()):
            assert not torch.allclose(final_values[:-1][at[:-1]], values[1:-1][at[:-1]], atol=1e-3)
        seen.append(int(at.sum()))
        return real(rewards, values, terminated, truncated, final_values, **kw)
    real = mod.gae
    monkeypatch.setattr(mod, "Policy", Policy)
    monkeypatch.setattr(mod, "Environment", Environment)
    monkeypatch.setattr(mod, "gae", gae)
    mod.train("gaussian", 32, n_envs=64, n_agents=3, steps=30, iterations=4, epochs=1,
              log=lambda line: None)
    assert sum(seen) > 0  # 120 steps, of which the 100th is the limit


def test_the_reward_rises():
    """Agents that move at random earn about -0.01 a step; ones that head for their goals ten times
    that, the other way."""
    rewards = example().train("gaussian", 32, iterations=45, log=lambda line: None)
    assert sum(rewards[-5:]) / 5 > sum(rewards[:5]) / 5 + 0.05
