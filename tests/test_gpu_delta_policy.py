"""Layer norm, delta rule and sampling together: a policy acting step by step against
the same policy over the whole rollout, its gradients against the plain forms, and
an actor that draws with cuts and a learner on the packed RL env."""

from __future__ import annotations

import pytest
import torch
from torch.nn import functional as F

from . import _policy_ref as ref
from .conftest import require_gpu
from .test_gpu_delta_rule import _plain as plain_delta

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu():
    require_gpu()


def _policy(dtype, dim=64):
    from gbxcule_amd.rl.memory import MemoryPolicy

    torch.manual_seed(4)
    policy = MemoryPolicy(8, dim=dim, blocks=2, dtype=dtype, memory="delta").cuda()
    with torch.no_grad():
        policy.heads.normal_(std=dim**-0.5)
    return policy


def test_steps_equal_the_rollout():
    """In 32 bits both forms compute the same sums in another order: about 100
    roundings of 2^-24 through two blocks, of values up to 10."""
    policy = _policy(torch.float32)
    steps, envs = 37, 13
    frames = torch.randint(0, 256, (steps, envs, 1, 72, 20), dtype=torch.uint8, device="cuda")
    resets = torch.rand(steps, envs, device="cuda") < 0.1
    state = policy.initial_state(envs)
    for s in state:
        s.window.normal_()
        s.scan.normal_(std=0.3)
    with torch.no_grad():
        logits, values = policy(frames, state, resets)
        for t in range(steps):
            one, value = policy.step(frames[t], state, resets[t])
            torch.testing.assert_close(one, logits[t], rtol=0, atol=1e-4)
            torch.testing.assert_close(value, values[t], rtol=0, atol=1e-4)


@pytest.mark.parametrize("share", [1, 2])
def test_gradients_of_a_block(share):
    from gbxcule_amd.rl.memory import BlockState, DeltaBlock

    torch.manual_seed(5)
    steps, envs, dim = 23, 3, 40
    block = DeltaBlock(dim, heads=2, keys=24, values=16, share=share, dtype=torch.float32).cuda()
    with torch.no_grad():
        block.norm.normal_(1.0, 0.2), block.norm_bias.normal_(std=0.2), block.head_norm.normal_(1.0, 0.2)
    hidden, stream = (torch.randn(steps, envs, dim, device="cuda", requires_grad=True) for _ in range(2))
    resets = torch.rand(steps, envs, device="cuda") < 0.1
    state = BlockState(*(torch.randn_like(t) * 0.3 for t in block.initial_state(envs)))
    weight = torch.randn(steps, envs, dim, device="cuda")
    out, kept = block(hidden, stream, state, resets)
    leaves = [hidden, stream, *block.parameters()]
    got = torch.autograd.grad((out * weight).sum() + (kept * weight).sum(), leaves)

    wide = {name: ref.f64(p) for name, p in block.named_parameters()}
    h, s = ref.f64(hidden), ref.f64(stream)
    total = h + s
    total = total + (total.detach().float().double() - total.detach())  # the stream's type
    c = total - total.mean(-1, keepdim=True)
    y = c / torch.sqrt((c * c).mean(-1, keepdim=True) + 1e-5) * wide["norm"] + wide["norm_bias"]
    x, z, dt, beta = (y @ wide["entry"].T).split([block.inner, 32, 2, 2], dim=-1)
    g = -torch.exp(wide["log_rate"]) * F.softplus(dt + wide["dt_bias"])
    x, _ = ref.causal_conv(x, wide["conv"], None, ref.f64(state.window), resets.cpu(), True)
    y, _ = plain_delta(*block._heads(x), g, torch.sigmoid(beta), ref.f64(state.scan), resets.cpu())
    y, _ = ref.rms_norm(y, wide["head_norm"], None, 1e-6, torch.float32)
    want_out = (y.flatten(-2) * F.silu(z)) @ wide["exit"].T
    ref.check(out, want_out, 400, "output")
    want = torch.autograd.grad((want_out * weight.cpu()).sum() + (total * weight.cpu()).sum(), [h, s, *wide.values()])
    names = ["hidden", "stream", *wide]
    for a, b, name in zip(got, want, names):
        # four operators and two products, each some hundred 32-bit roundings there and back, and sums over 69 rows
        ref.check(a, b, 2000, f"gradient of {name}")


@pytest.mark.parametrize("ladder", [False, True])
def test_rollout_and_learner(ladder, carts):
    from gbxcule_amd.rl import AdamW, PackedPixelEnv, RolloutBuffer, collect_rollout
    from gbxcule_amd.rl.memory import MemoryActor, learn

    n, steps = 48, 19

    def reward(env, pixels, senses):
        return pixels[:, 0, 0, 0].float() / 255, torch.arange(n, device="cuda") % 7 == env._episode_step % 7

    env = PackedPixelEnv(carts["c3"], num_envs=n, frames_per_step=2, reward_fn=reward)
    try:
        env.reset(seed=0)
        rollout = RolloutBuffer(steps=steps, num_envs=n, stack_k=1, obs_format="packed2", obs_steps=steps + 1)
        policy = _policy(torch.bfloat16)
        before = [p.detach().clone() for p in policy.parameters()]
        opt = AdamW(policy.parameters(), lr=3e-3, state_bits=8)
        heat = torch.linspace(0.0, 2.0, n, device="cuda")
        actor = MemoryActor(policy, n, rollout, sampling={"temperature": heat, "top_k": 5, "top_p": 0.9} if ladder else {})
        for k in range(2):
            if k:
                actor.begin_rollout()
            last = collect_rollout(env, actor, rollout)
            assert bool(rollout.dones.any()) and torch.isfinite(rollout.logprobs).all()
            assert int(rollout.actions.min()) >= 0 and int(rollout.actions.max()) < 8
            with torch.no_grad():
                logits, values = policy(rollout.obs[:steps], actor.first_state, actor.resets())
            if ladder:  # the coldest env takes its likeliest action, with certainty
                assert not rollout.logprobs[:, 0].any()
                likeliest = logits[:, 0].max(-1).values - logits[:, 0].gather(-1, rollout.actions[:, :1].long()).squeeze(-1)
                assert float(likeliest.max()) < 0.05  # the actor's and the learner's logits differ by 16-bit rounding
            else:
                logp = torch.log_softmax(logits, -1).gather(-1, rollout.actions.long().unsqueeze(-1)).squeeze(-1)
                assert float((logp - rollout.logprobs).abs().mean()) < 0.05
            losses = learn(actor, opt, last, passes=3)
            assert all(torch.isfinite(v) for v in losses)
        assert any(not torch.equal(a, b) for a, b in zip(before, policy.parameters()))
        assert all(torch.isfinite(p).all() for p in policy.parameters())
    finally:
        env.close()


def test_refusals():
    from gbxcule_amd.rl.memory import DeltaBlock, MemoryActor, MemoryPolicy

    with pytest.raises(ValueError, match="memory"):
        MemoryPolicy(8, memory="attention")
    with pytest.raises(ValueError, match="share"):
        DeltaBlock(32, heads=3, share=2)
    policy = _policy(torch.bfloat16)
    with pytest.raises(ValueError, match="fp8"):
        MemoryActor(policy, 4, None, fp8=True)


def test_an_env_whose_state_is_not_finite_plays_an_action(carts):
    """Its logits are NaN, so nothing can be drawn from them: it plays on, and rollout and loss say so."""
    from gbxcule_amd.rl import AdamW, PackedPixelEnv, RolloutBuffer, collect_rollout
    from gbxcule_amd.rl.memory import MemoryActor, learn

    n, steps = 8, 5
    env = PackedPixelEnv(carts["c3"], num_envs=n, frames_per_step=2)
    try:
        env.reset(seed=0)
        rollout = RolloutBuffer(steps=steps, num_envs=n, stack_k=1, obs_format="packed2", obs_steps=steps + 1)
        policy = _policy(torch.bfloat16)
        actor = MemoryActor(policy, n, rollout, sampling={"temperature": 0.9})
        actor.begin_rollout(torch.zeros(n, dtype=torch.bool, device="cuda"))
        for s in actor.state:
            s.scan[2] = float("nan")
        actor.begin_rollout(actor.starts)
        last = collect_rollout(env, actor, rollout)
        assert int(rollout.actions.min()) >= 0 and int(rollout.actions.max()) < 8
        bad = torch.isnan(rollout.logprobs)
        assert bad[:, 2].all() and int(bad.sum()) == steps
        (loss,) = learn(actor, AdamW(policy.parameters(), lr=1e-3), last, passes=1)
        assert torch.isnan(loss)
    finally:
        env.close()
