"""A policy that remembers its episode, built from the operators of ``ops``,
with the actor and the learner around ``collect_rollout``.

``python -m gbxcule_amd.rl.memory`` plays the synthetic PPU cart and learns
from a few rollouts.

The policy reads packed frames, carries a selective state space through the
steps of an episode and returns action logits and a value.  The actor holds one
state per env and makes one step of all envs at a time, with the projection at
each block's entry in 8 bits on request; the learner reads the same rollout as
``[T, N]`` with the episode starts, from the state the rollout began with.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch
from torch import nn
from torch.nn import functional as F

from ..abi import DOWNSAMPLE_H, DOWNSAMPLE_W
from .ops import causal_conv, causal_conv_step, rms_norm, rms_norm_fp8, selective_scan, selective_scan_step
from .packed import unpack_2bpp_u8

E4M3_MAX = 448.0


class BlockState(NamedTuple):
    """What a block carries: the convolution's last inputs ``[N, 3, inner]`` and
    the scan's state ``[N, inner, states]``."""

    window: torch.Tensor
    scan: torch.Tensor


class MemoryBlock(nn.Module):
    """norm -> projection -> causal convolution -> selective scan -> projection.
    ``hidden`` is what the block before adds to the ``stream``."""

    def __init__(self, dim: int, states: int = 16, width: int = 4, dtype=torch.bfloat16) -> None:
        super().__init__()
        inner, rank = 2 * dim, -(-dim // 16)
        self.inner, self.states, self.rank, self.width = inner, states, rank, width
        self.norm = nn.Parameter(torch.ones(dim))
        self.entry = nn.Parameter(torch.randn(2 * inner, dim, dtype=dtype) * dim**-0.5)
        self.conv = nn.Parameter(torch.randn(inner, width) * width**-0.5)
        self.conv_bias = nn.Parameter(torch.zeros(inner))
        self.choose = nn.Parameter(torch.randn(rank + 2 * states, inner, dtype=dtype) * inner**-0.5)
        self.dt = nn.Parameter(torch.randn(inner, rank, dtype=dtype) * rank**-0.5)
        size = torch.exp(torch.rand(inner) * math.log(100.0) + math.log(1e-3))  # steps of 0.001 to 0.1
        self.dt_bias = nn.Parameter(size + torch.log(-torch.expm1(-size)))
        self.log_rate = nn.Parameter(torch.log(torch.arange(1.0, states + 1)).repeat(inner, 1))
        self.skip = nn.Parameter(torch.ones(inner))
        self.exit = nn.Parameter(torch.randn(dim, inner, dtype=dtype) * inner**-0.5)

    def initial_state(self, envs: int) -> BlockState:
        like = self.entry
        return BlockState(like.new_zeros(envs, self.width - 1, self.inner),
                          self.skip.new_zeros(envs, self.inner, self.states))  # fmt: skip

    def _choices(self, x):
        """dt, B and C of a step, from the convolved input."""
        dt, b, c = F.linear(x, self.choose).split([self.rank, self.states, self.states], dim=-1)
        return F.linear(dt, self.dt), b, c

    def forward(self, hidden, stream, state: BlockState, resets):
        """A rollout: ``[T, N, dim]`` and ``resets`` ``[T, N]``; the state stays
        as it is.  Returns ``(hidden, stream)``."""
        y, stream = (rms_norm(hidden, self.norm), hidden) if stream is None else rms_norm(hidden, self.norm, stream)
        x, gate = F.linear(y, self.entry).chunk(2, dim=-1)
        x, _ = causal_conv(x, self.conv, self.conv_bias, state=state.window, resets=resets)
        dt, b, c = self._choices(x)
        y, _ = selective_scan(x, dt, -torch.exp(self.log_rate), b, c, self.skip, gate, dt_bias=self.dt_bias,
                              state=state.scan, resets=resets)  # fmt: skip
        return F.linear(y, self.exit), stream

    def step(self, hidden, stream, state: BlockState, resets, entry_fp8=None):
        """One step of all envs, ``[N, dim]``; the state moves on in place.
        ``entry_fp8``: the entry projection of ``quantized_entry``."""
        if entry_fp8 is None:
            y, stream = (rms_norm(hidden, self.norm), hidden) if stream is None else rms_norm(hidden, self.norm, stream)
            both = F.linear(y, self.entry)
        else:
            q, scale, *kept = rms_norm_fp8(hidden, self.norm, stream)
            stream = kept[0] if kept else hidden
            weight, weight_scale = entry_fp8
            rows = F.ScalingType.RowWise
            both = F.scaled_mm(q, weight.t(), scale.unsqueeze(-1), rows, weight_scale, rows, output_dtype=hidden.dtype)
        x, gate = both.chunk(2, dim=-1)
        x = causal_conv_step(x, self.conv, self.conv_bias, state.window, resets=resets)
        dt, b, c = self._choices(x)
        y = selective_scan_step(x, dt, -torch.exp(self.log_rate), b, c, self.skip, gate, state=state.scan,
                                dt_bias=self.dt_bias, resets=resets)  # fmt: skip
        return F.linear(y, self.exit), stream

    def quantized_entry(self):
        """The entry projection in 8 bits with a scale for each output."""
        w = self.entry.float()
        scale = w.abs().amax(1).clamp_min(1e-30) / E4M3_MAX
        return (w / scale[:, None]).to(torch.float8_e4m3fn), scale.unsqueeze(0)


class MemoryPolicy(nn.Module):
    """Packed frames ``[..., 1, 72, 20]`` -> action logits and values."""

    def __init__(self, num_actions: int, *, dim: int = 256, blocks: int = 2, states: int = 16, dtype=torch.bfloat16) -> None:
        super().__init__()
        pixels = DOWNSAMPLE_H * DOWNSAMPLE_W
        self.dtype = dtype
        self.eye = nn.Parameter(torch.randn(dim, pixels, dtype=dtype) * pixels**-0.5)
        self.blocks = nn.ModuleList(MemoryBlock(dim, states, dtype=dtype) for _ in range(blocks))
        self.norm = nn.Parameter(torch.ones(dim))
        self.heads = nn.Parameter(torch.zeros(num_actions + 1, dim, dtype=dtype))

    def initial_state(self, envs: int) -> list[BlockState]:
        return [b.initial_state(envs) for b in self.blocks]

    def _see(self, frames):
        shades = unpack_2bpp_u8(frames).flatten(-3)
        return F.linear(shades.to(self.dtype) / 1.5 - 1.0, self.eye)

    def _answer(self, hidden, stream):
        y, _ = rms_norm(hidden, self.norm, stream)
        out = F.linear(y, self.heads).float()
        return out[..., :-1], out[..., -1]

    def forward(self, frames, state: list[BlockState], resets):
        """A rollout ``[T, N, 1, 72, 20]`` from ``state``: logits ``[T, N, actions]``, values ``[T, N]``."""
        hidden, stream = self._see(frames), None
        for block, s in zip(self.blocks, state):
            hidden, stream = block(hidden, stream, s, resets)
        return self._answer(hidden, stream)

    @torch.no_grad()
    def step(self, frames, state: list[BlockState], resets, entries_fp8=None):
        """One step of all envs ``[N, 1, 72, 20]``; ``state`` moves on in place."""
        hidden, stream = self._see(frames), None
        for k, (block, s) in enumerate(zip(self.blocks, state)):
            hidden, stream = block.step(hidden, stream, s, resets, None if entries_fp8 is None else entries_fp8[k])
        return self._answer(hidden, stream)


class MemoryActor:
    """The ``policy`` argument of ``collect_rollout``: keeps the envs' states and
    takes the episode starts from the rollout's rows of the step before."""

    def __init__(self, policy: MemoryPolicy, num_envs: int, rollout, *, fp8: bool = False) -> None:
        self.policy, self.rollout, self.fp8 = policy, rollout, fp8
        self.state = policy.initial_state(num_envs)
        self.begin_rollout(torch.ones(num_envs, dtype=torch.bool, device=policy.eye.device))

    @torch.no_grad()
    def begin_rollout(self, starts=None) -> None:
        """Before each rollout: remembers the state and the episode starts it
        begins with (default: where the last rollout's last step ended one)."""
        self.starts = self.rollout.dones[-1].clone() if starts is None else starts
        self.first_state = [BlockState(*(t.clone() for t in s)) for s in self.state]
        self.entries = [b.quantized_entry() for b in self.policy.blocks] if self.fp8 else None

    def __call__(self, frames):
        t = self.rollout.step
        resets = self.starts if t == 0 else self.rollout.dones[t - 1]
        logits, values = self.policy.step(frames, self.state, resets, self.entries)
        logp = torch.log_softmax(logits, -1)
        noise = -torch.log(-torch.log(torch.rand_like(logp).clamp_min(1e-20)).clamp_min(1e-20))
        actions = (logp + noise).argmax(-1)
        return actions.to(torch.int32), values, logp.gather(-1, actions.unsqueeze(-1)).squeeze(-1)

    def resets(self):
        """Episode starts ``[T, N]`` of the rollout that was collected."""
        return torch.cat([self.starts.unsqueeze(0), self.rollout.dones[:-1]])


@torch.no_grad()
def advantages(rewards, dones, values, last_value, *, discount: float = 0.99, trace: float = 0.95):
    """Generalised advantages ``[T, N]``, cut where an episode ends."""
    out, run = torch.empty_like(rewards), torch.zeros_like(last_value)
    for t in range(rewards.shape[0] - 1, -1, -1):
        go = (~dones[t]).float()
        delta = rewards[t] + discount * last_value * go - values[t]
        run = delta + discount * trace * go * run
        out[t], last_value = run, values[t]
    return out


def learn(actor: MemoryActor, optimizer, last_frames, *, passes: int = 2, clip: float = 0.2, max_norm: float = 1.0) -> list:
    """Clipped policy-gradient passes over the collected rollout; returns the
    losses as device scalars (nothing here synchronises)."""
    policy, r = actor.policy, actor.rollout
    # the value after the last step, from a copy of the states the rollout ended with
    state = [BlockState(*(t.clone() for t in s)) for s in actor.state]
    _, last_value = policy.step(last_frames, state, r.dones[-1], actor.entries)
    gain = advantages(r.rewards, r.dones, r.values, last_value)
    target = gain + r.values
    gain = (gain - gain.mean()) / (gain.std() + 1e-6)
    frames, resets, actions = r.obs[: r.steps], actor.resets(), r.actions.long().unsqueeze(-1)
    losses = []
    for _ in range(passes):
        logits, values = policy(frames, actor.first_state, resets)
        logp = torch.log_softmax(logits, -1)
        ratio = torch.exp(logp.gather(-1, actions).squeeze(-1) - r.logprobs)
        gained = torch.minimum(ratio * gain, ratio.clamp(1 - clip, 1 + clip) * gain)
        entropy = -(logp.exp() * logp).sum(-1)
        loss = -gained.mean() + 0.5 * (values - target).square().mean() - 0.01 * entropy.mean()
        optimizer.zero_grad()
        loss.backward()
        norms = torch._foreach_norm([p.grad.float() for p in policy.parameters()])
        scale = (max_norm / (torch.stack(norms).norm() + 1e-6)).clamp_max(1.0)
        optimizer.step(grad_scale=scale)
        losses.append(loss.detach())
    return losses


def main(num_envs: int = 1024, steps: int = 32, rollouts: int = 4) -> None:
    import time

    from ..carts.synth import cart_c3
    from . import AdamW, PackedPixelEnv, RolloutBuffer, collect_rollout, packed_l1_distance

    goal = torch.randint(0, 256, (1, DOWNSAMPLE_H, 20), dtype=torch.uint8, device="cuda")

    def reward(env, pixels, senses):
        return 1.0 - packed_l1_distance(pixels, goal), torch.rand(env.num_envs, device="cuda") < 0.01

    torch.manual_seed(0)
    env = PackedPixelEnv(cart_c3(2), num_envs=num_envs, reward_fn=reward)
    env.reset(seed=0)
    rollout = RolloutBuffer(steps=steps, num_envs=num_envs, stack_k=1, obs_format="packed2", obs_steps=steps + 1)
    policy = MemoryPolicy(env.num_actions).cuda()
    optimizer = AdamW(policy.parameters(), lr=1e-3, state_bits=8)
    actor = MemoryActor(policy, num_envs, rollout, fp8=True)
    for k in range(rollouts):
        if k:
            actor.begin_rollout()
        torch.cuda.synchronize()
        began = time.perf_counter()
        last = collect_rollout(env, actor, rollout)
        torch.cuda.synchronize()
        played = time.perf_counter()
        losses = [round(float(v), 4) for v in learn(actor, optimizer, last)]
        print(f"rollout {k}: {num_envs * steps / (played - began):,.0f} env-steps/s, losses {losses}, "
              f"learner {time.perf_counter() - played:.3f} s", flush=True)  # fmt: skip
    env.close()


if __name__ == "__main__":
    main()
