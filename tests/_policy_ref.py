"""Plain 64-bit forms of the policy operators, step by step on the CPU, with
gradients from torch's autograd, and the tolerances that the kernels' outputs
are held to."""

from __future__ import annotations

import torch

# One rounding of the output type is half a unit in the last place, and a value
# next to a rounding boundary may go to the other side of it: one unit.
UNIT = {torch.float32: 2.0**-23, torch.bfloat16: 2.0**-7, torch.float16: 2.0**-10}
# The smallest step of float16 is absolute: its subnormal unit.
FLOOR = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0**-24}


def check(got, want, roundings: int, what: str = "") -> None:
    """``roundings``: 32-bit roundings that a value may go through, each of the
    size of the largest value; then one rounding to got's type."""
    want = want.detach().cpu().double()
    got = got.detach().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    big = float(want[torch.isfinite(want)].abs().max()) if want.numel() and torch.isfinite(want).any() else 0.0
    atol = roundings * 2.0**-23 * big + FLOOR[got.dtype] + 1e-30
    torch.testing.assert_close(got.double(), want, rtol=UNIT[got.dtype], atol=atol, equal_nan=True, msg=lambda m: f"{what}: {m}")


def f64(t):
    return None if t is None else t.detach().cpu().double().requires_grad_(t.requires_grad)


def rms_norm(x, weight, residual, eps, stream_type):
    """(y, s); s is rounded to the stream's type, with the gradient of the sum."""
    s = x
    if residual is not None:
        s = x + residual
        s = s + (s.detach().to(stream_type).double() - s.detach())
    return s / torch.sqrt((s * s).mean(-1, keepdim=True) + eps) * weight, s


def causal_conv(x, weight, bias, state, resets, silu):
    steps, envs, dim = x.shape
    width = weight.shape[1]
    window = list(state.unbind(1)) if state is not None else [torch.zeros(envs, dim, dtype=x.dtype)] * (width - 1)
    out = []
    for t in range(steps):
        if resets is not None:
            window = [torch.where(resets[t, :, None] != 0, 0.0, w) for w in window]
        window = [*window, x[t]]
        pre = sum(w * weight[:, i] for i, w in enumerate(window))
        if bias is not None:
            pre = pre + bias
        out.append(pre * torch.sigmoid(pre) if silu else pre)
        window = window[1:]
    return torch.stack(out), torch.stack(window, 1)


def selective_scan(x, dt, A, B, C, D, z, dt_bias, softplus, state, resets):
    steps, envs, dim = x.shape
    groups = B.shape[2]
    h = state if state is not None else torch.zeros(envs, *A.shape, dtype=torch.float64)
    delta = dt if dt_bias is None else dt + dt_bias
    if softplus:
        delta = torch.logaddexp(delta, torch.zeros((), dtype=torch.float64))
    wide = lambda t: t.repeat_interleave(dim // groups, dim=1)  # noqa: E731
    out = []
    for t in range(steps):
        if resets is not None:
            h = torch.where(resets[t, :, None, None] != 0, 0.0, h)
        h = torch.exp(delta[t, ..., None] * A) * h + (delta[t] * x[t])[..., None] * wide(B[t])
        y = (h * wide(C[t])).sum(-1)
        if D is not None:
            y = y + D * x[t]
        if z is not None:
            y = y * z[t] * torch.sigmoid(z[t])
        out.append(y)
    return torch.stack(out), h


def noise(index, key):
    h = ((index ^ key) * 0x9E3779B9) & 0xFFFFFFFF
    h = h ^ (h >> 16)
    h = (h * 0x6A09E667) & 0xFFFFFFFF
    return h ^ (h >> 15)
