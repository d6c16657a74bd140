"""The operators together: a policy acting step by step, in 16 and in 8 bits,
against the same policy over the whole rollout, and a learner on the packed RL
env."""

from __future__ import annotations

import pytest
import torch

from .conftest import require_gpu

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu():
    require_gpu()


def _policy(dtype, dim=64):
    from gbxcule_amd.rl.memory import MemoryPolicy

    torch.manual_seed(3)
    policy = MemoryPolicy(8, dim=dim, blocks=2, dtype=dtype).cuda()
    with torch.no_grad():
        policy.heads.normal_(std=dim**-0.5)
    return policy


def test_steps_equal_the_rollout():
    """In 32 bits both forms compute the same sums in another order: about 100
    roundings of 2^-24 through two blocks, of values up to 10."""
    policy = _policy(torch.float32)
    steps, envs = 21, 13
    frames = torch.randint(0, 256, (steps, envs, 1, 72, 20), dtype=torch.uint8, device="cuda")
    resets = torch.rand(steps, envs, device="cuda") < 0.15
    state = policy.initial_state(envs)
    for s in state:
        s.window.normal_()
        s.scan.normal_()
    with torch.no_grad():
        logits, values = policy(frames, state, resets)
        for t in range(steps):
            one, value = policy.step(frames[t], state, resets[t])
            torch.testing.assert_close(one, logits[t], rtol=0, atol=1e-4)
            torch.testing.assert_close(value, values[t], rtol=0, atol=1e-4)


def test_actor_in_8_bits_is_near():
    """e4m3 rounds each product's operands by up to 2^-4, about 3% at random: the
    logits of two blocks move by a few per cent of their size."""
    policy = _policy(torch.bfloat16, dim=128)
    envs = 300
    frames = torch.randint(0, 256, (envs, 1, 72, 20), dtype=torch.uint8, device="cuda")
    resets = torch.ones(envs, dtype=torch.bool, device="cuda")
    entries = [b.quantized_entry() for b in policy.blocks]
    full, _ = policy.step(frames, policy.initial_state(envs), resets)
    small, _ = policy.step(frames, policy.initial_state(envs), resets, entries)
    assert float((small - full).norm() / full.norm()) < 0.15
    assert float((small - full).norm() / full.norm()) > 1e-4  # the 8-bit path ran


@pytest.mark.parametrize("bits, fp8", [(32, False), (8, True)])
def test_rollout_and_learner(bits, fp8, carts):
    from gbxcule_amd.rl import AdamW, PackedPixelEnv, RolloutBuffer, collect_rollout
    from gbxcule_amd.rl.memory import MemoryActor, learn

    n, steps = 48, 9

    def reward(env, pixels, senses):
        return pixels[:, 0, 0, 0].float() / 255, torch.arange(n, device="cuda") % 7 == env._episode_step % 7

    env = PackedPixelEnv(carts["c3"], num_envs=n, frames_per_step=2, reward_fn=reward)
    try:
        env.reset(seed=0)
        rollout = RolloutBuffer(steps=steps, num_envs=n, stack_k=1, obs_format="packed2", obs_steps=steps + 1)
        policy = _policy(torch.bfloat16)
        before = [p.detach().clone() for p in policy.parameters()]
        opt = AdamW(policy.parameters(), lr=3e-3, state_bits=bits)
        actor = MemoryActor(policy, n, rollout, fp8=fp8)
        for k in range(2):
            if k:
                actor.begin_rollout()
            last = collect_rollout(env, actor, rollout)
            assert bool(rollout.dones.any()) and torch.isfinite(rollout.logprobs).all()
            resets = actor.resets()
            assert resets.shape == (steps, n) and torch.equal(resets[1:], rollout.dones[:-1])
            # what the learner computes is what the actor did, to 16-bit (8-bit) rounding
            with torch.no_grad():
                logits, values = policy(rollout.obs[:steps], actor.first_state, resets)
            logp = torch.log_softmax(logits, -1).gather(-1, rollout.actions.long().unsqueeze(-1)).squeeze(-1)
            assert float((logp - rollout.logprobs).abs().mean()) < (0.2 if fp8 else 0.05)
            losses = learn(actor, opt, last, passes=12)
            assert all(torch.isfinite(v) for v in losses) and float(losses[-1]) < float(losses[0])
        assert any(not torch.equal(a, b) for a, b in zip(before, policy.parameters()))
        assert all(torch.isfinite(p).all() for p in policy.parameters())
    finally:
        env.close()
