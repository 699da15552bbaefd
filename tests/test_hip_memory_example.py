"""The training example's policy with a memory and its imitation: that they run, that acting step by
step and training on the rollout see the same, and the gradients of a whole update against float64."""

import importlib.util
import math
from pathlib import Path

import pytest
import torch

from swarp_amd import AdamW, categorical_policy_loss, gae, linear_cross_entropy

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def example():
    path = Path(__file__).resolve().parents[1] / "examples" / "train_navigation.py"
    spec = importlib.util.spec_from_file_location("train_navigation", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("head,memory,clone,bits", [("categorical", 4, 3, 32), ("categorical", 0, 2, 8),
                                                    ("gaussian", 2, 0, 32)])
def test_it_runs(head, memory, clone, bits):
    lines = []
    rewards = example().train(head, bits, n_envs=48, n_agents=3, steps=40, iterations=3, epochs=2,
                              memory=memory, clone=clone, log=lines.append)
    assert len(rewards) == clone + 3 and all(math.isfinite(r) for r in rewards)
    assert sum("imitation" in x for x in lines) == clone and not any("nan" in x for x in lines)


def test_the_expert_points_to_the_goal():
    mod = example()
    policy = mod.Policy(9, 2, "categorical").to(DEV)
    obs = torch.zeros(10, 9, device=DEV)
    obs[:9, 7:9] = policy.moves * 2
    obs[9, 7:9] = 0.01
    assert mod.expert(policy, obs).tolist() == [0, 1, 2, 3, 4, 5, 6, 7, 8, 8]


def test_only_moves_are_imitated():
    with pytest.raises(ValueError, match="imitated"):
        example().train("gaussian", clone=1)


def plain_memory(m, h, state, starts):
    """Memory.forward step by step, in h's type."""
    out = []
    for t in range(h.shape[0]):
        q, k, v = m.qkv(h[t]).unflatten(-1, (3, m.heads, -1)).unbind(-3)
        keep = torch.exp(m.log_decay)[:, None, None] * ~starts[t][:, None, None, None, None]
        state = keep * state + k[..., :, None] * v[..., None, :]
        o = (q[..., None, :] @ state)[..., 0, :] * q.shape[-1] ** -0.5
        out.append(h[t] + m.mix(o.flatten(-2)))
    return torch.stack(out)


def test_an_update_of_a_rollout():
    """Acting with the step form, then advantages, the policy's and the imitation's loss and AdamW on the
    rollout.  Everything is float32: sums of some hundreds of terms behind one another, of which 1e-4
    of the largest is far from what a mistake would make."""
    mod = example()
    torch.manual_seed(3)
    T, E, A = 21, 7, 3
    policy = mod.Policy(11, 2, "categorical", 64, 4).to(DEV)
    with torch.no_grad():
        policy.out.weight.mul_(50.0)
    obs = torch.randn(T, E, A, 11, device=DEV)
    starts = torch.rand(T, E, device=DEV) < 0.15
    state = torch.randn_like(policy.memory.empty(E, A))
    acted, now = [], state.clone()
    for t in range(T):
        seen = now.clone()
        value = policy.value_after(obs[t], now, starts[t])
        assert torch.equal(now, seen)
        acted.append(policy.act(obs[t], now, starts[t]))
        assert torch.equal(value, acted[-1][3])
    choice, _, logp, value = (torch.stack(x) for x in zip(*acted))
    scanned = policy(obs, state, starts)
    assert torch.allclose(scanned[1], value, rtol=1e-4, atol=1e-4)
    again = torch.log_softmax(scanned[0], -1).gather(-1, choice[..., None])[..., 0]
    assert torch.allclose(again, logp, rtol=1e-4, atol=1e-4)

    reward = torch.randn(T, E, A, device=DEV)
    done = torch.rand(T, E, device=DEV) < 0.15
    adv, returns = gae(reward, torch.cat([value, value[-1:]]), done)
    moves = torch.randint(0, 9, (T, E, A), device=DEV)

    def losses(p, o, plain):
        if not plain:
            h = p.features(o, state, starts)
            out, v = p.out(h), p.value(h)[..., 0]
            pg = categorical_policy_loss(out, choice, logp, adv, entropy_coef=0.01).loss
            same = linear_cross_entropy(h, p.out.weight, moves, p.out.bias).loss
        else:
            h = plain_memory(p.memory, p.trunk(o), state.double(), starts)
            out, v = p.out(h), p.value(h)[..., 0]
            all_p = torch.log_softmax(out, -1)
            ratio = torch.exp(all_p.gather(-1, choice[..., None])[..., 0] - logp.double())
            pg = -torch.minimum(ratio * adv, ratio.clamp(0.8, 1.2) * adv).mean()
            pg = pg + 0.01 * (all_p.exp() * all_p).sum(-1).mean()
            same = -all_p.gather(-1, moves[..., None]).mean()
        return pg + 0.5 * (v - returns).square().mean() + same
    exact = mod.Policy(11, 2, "categorical", 64, 4).to(DEV)
    exact.load_state_dict(policy.state_dict())
    exact = exact.double()
    exact.memory.log_decay.copy_(policy.memory.log_decay)
    names = [n for n, _ in policy.named_parameters()]
    got = losses(policy, obs, False)
    want = losses(exact, obs.double(), True)
    assert abs(float(got) - float(want)) < 1e-4 * max(1.0, abs(float(want)))
    got.backward()
    want.backward()
    for n, p, e in zip(names, policy.parameters(), exact.parameters()):
        assert float((p.grad - e.grad).abs().max()) <= 1e-4 * float(e.grad.abs().max()), n
    before = [p.detach().clone() for p in policy.parameters()]
    AdamW(policy.parameters(), lr=1e-3, max_grad_norm=0.5).step()
    assert all(not torch.equal(p, b) and bool(p.isfinite().all()) for p, b in zip(policy.parameters(), before))
