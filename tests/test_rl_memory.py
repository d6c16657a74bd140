"""The actor and the learner of ``gbxcule_amd.rl.memory`` around a policy whose
logits are given, on the CPU: what the actor stores of a draw, and what the
learner makes of it."""

from __future__ import annotations

import math
import types

import pytest
import torch
from torch import nn

from gbxcule_amd.rl import RolloutBuffer, memory

STEPS, ENVS, ACTIONS = 5, 6, 4


class GivenPolicy(nn.Module):
    """Logits and values of each step and env as parameters."""

    memory = "delta"

    def __init__(self) -> None:
        super().__init__()
        gen = torch.Generator().manual_seed(1)
        self.logits = nn.Parameter(torch.randn(STEPS, ENVS, ACTIONS, generator=gen))
        self.values = nn.Parameter(torch.randn(STEPS, ENVS, generator=gen))
        self.eye = torch.zeros(1)
        self.blocks = nn.ModuleList()
        self.at = 0

    def initial_state(self, envs):
        return []

    def forward(self, frames, state, resets):
        return self.logits, self.values

    @torch.no_grad()
    def step(self, frames, state, resets, entries=None):
        k = min(self.at, STEPS - 1)
        self.at += 1
        return self.logits[k].detach(), self.values[k].detach()


class Kept:
    """An optimizer that moves nothing and keeps the gradients of each step."""

    def __init__(self, policy) -> None:
        self.policy, self.seen = policy, []

    def zero_grad(self) -> None:
        self.policy.zero_grad()

    def step(self, grad_scale) -> None:
        self.seen.append([p.grad.clone() for p in self.policy.parameters()])


def _draw(logits, uniform, *, temperature=1.0, **_):
    """``sample_actions`` on the CPU, with temperatures alone."""
    heat = torch.as_tensor(temperature, dtype=torch.float64).expand(len(logits)).unsqueeze(-1)
    sharp = torch.log_softmax(logits.double() / heat.clamp_min(1e-6), -1)
    action = (sharp.exp().cumsum(-1) <= uniform.double().unsqueeze(-1)).sum(-1).clamp_max(logits.shape[-1] - 1)
    logp = sharp.gather(-1, action.unsqueeze(-1)).squeeze(-1)
    nothing = torch.isnan(logits).all(-1)
    return torch.where(nothing, -1, action).int(), torch.where(nothing, math.nan, logp).float()


def _played(monkeypatch, policy, sampling):
    monkeypatch.setattr(memory, "sample_actions", _draw)
    torch.manual_seed(2)
    rollout = RolloutBuffer(steps=STEPS, num_envs=ENVS, stack_k=1, obs_format="packed2", device="cpu", obs_steps=STEPS + 1)
    actor = memory.MemoryActor(policy, ENVS, rollout, sampling=sampling)
    rollout.reset()
    for t in range(STEPS):
        actions, values, logp = actor(rollout.obs_slot(t))
        rollout.set_step_fields(t, actions, torch.randn(ENVS), torch.zeros(ENVS, dtype=torch.bool), values, logp)
    return actor, rollout


def test_an_env_with_nothing_to_draw_from_plays_an_action(monkeypatch):
    """A policy that has diverged: the sampler's -1 is no action, and the learner reads logits by the actions."""
    policy = GivenPolicy()
    with torch.no_grad():
        policy.logits[:, 2] = math.nan
    actor, rollout = _played(monkeypatch, policy, {})
    assert int(rollout.actions.min()) >= 0 and int(rollout.actions.max()) < ACTIONS
    assert torch.isnan(rollout.logprobs[:, 2]).all() and torch.isfinite(rollout.logprobs[:, :2]).all()
    (loss,) = memory.learn(actor, Kept(policy), rollout.obs_slot(STEPS), passes=1)
    assert torch.isnan(loss)  # as with the default actor: it shows


def _advantage(rollout):
    gain = memory.advantages(rollout.rewards, rollout.dones, rollout.values, rollout.values[-1])
    return (gain - gain.mean()) / (gain.std() + 1e-6)


@pytest.mark.parametrize("temperature", [0.0, 0.3, 1.0, 2.0])
def test_the_clip_is_around_the_policy_that_drew(monkeypatch, temperature):
    """The first pass's gradient is that of the weighted gains, with every ratio 1 and so no action
    clipped away: an env that always takes its likeliest action learns from the bad ones, too."""
    policy = GivenPolicy()
    actor, rollout = _played(monkeypatch, policy, {"temperature": temperature})
    kept = Kept(policy)
    memory.learn(actor, kept, rollout.obs_slot(STEPS), passes=1)
    logits = policy.logits.detach().double().requires_grad_()
    logp = torch.log_softmax(logits, -1)
    taken = logp.gather(-1, rollout.actions.long().unsqueeze(-1)).squeeze(-1)
    weight = torch.exp(taken.detach() - rollout.logprobs.double()).clamp_max(1.0)
    gain = _advantage(rollout).double()
    (-(weight * gain * taken).mean() + 0.01 * (logp.exp() * logp).sum(-1).mean()).backward()
    torch.testing.assert_close(kept.seen[0][0].double(), logits.grad, rtol=1e-4, atol=1e-6)
    if temperature == 0.0:
        assert bool(((taken.detach().exp() < 1 - 0.2) & (gain < 0)).any())  # which a clip around the draw's own 1 would drop


def test_an_actor_without_options_is_learned_from_as_before(monkeypatch):
    """The clip is around what the actor stored."""
    policy = GivenPolicy()
    actor, rollout = _played(monkeypatch, policy, None)
    rollout.logprobs.sub_(0.05)  # as 16-bit rounding may move them
    kept = Kept(policy)
    memory.learn(actor, kept, rollout.obs_slot(STEPS), passes=1, clip=0.01)
    logits = policy.logits.detach().double().requires_grad_()
    logp = torch.log_softmax(logits, -1)
    ratio = torch.exp(logp.gather(-1, rollout.actions.long().unsqueeze(-1)).squeeze(-1) - rollout.logprobs.double())
    gain = _advantage(rollout).double()
    gained = torch.minimum(ratio * gain, ratio.clamp(0.99, 1.01) * gain)
    (-gained.mean() + 0.01 * (logp.exp() * logp).sum(-1).mean()).backward()
    torch.testing.assert_close(kept.seen[0][0].double(), logits.grad, rtol=1e-4, atol=1e-6)


def test_policies_and_actors_from_before_the_options():
    """One that was saved whole, or a policy of a user's own, has no kind of memory and no options of a draw."""
    policy = memory.MemoryPolicy(ACTIONS, dim=16, blocks=1)
    policy.__dict__.pop("memory", None)
    rollout = RolloutBuffer(steps=STEPS, num_envs=ENVS, stack_k=1, obs_format="packed2", device="cpu", obs_steps=STEPS + 1)
    actor = memory.MemoryActor(policy, ENVS, rollout, fp8=True)
    assert policy.memory == "scan" and len(actor.entries) == 1
    actor.__dict__.pop("sampling", None)
    assert actor.sampling is None

    class Own(GivenPolicy):
        @property
        def memory(self):
            raise AttributeError("memory")

    assert memory.MemoryActor(Own(), ENVS, rollout, fp8=True).entries == []


def test_an_actor_of_a_users_own(monkeypatch):
    """What ``learn`` reads of it is what it read before there were options."""
    policy = GivenPolicy()
    actor, rollout = _played(monkeypatch, policy, None)
    names = ("policy", "rollout", "state", "first_state", "entries", "resets")
    own = types.SimpleNamespace(**{name: getattr(actor, name) for name in names})
    both = Kept(policy)
    for a in (actor, own):
        memory.learn(a, both, rollout.obs_slot(STEPS), passes=1)
    assert all(torch.equal(p, q) for p, q in zip(*both.seen))
