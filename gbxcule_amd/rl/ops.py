"""Operators of a policy that remembers an episode, as HIP kernels.

A memory block normalises its input (``rms_norm``), mixes the last few steps
of each env (``causal_conv``), carries a state along the steps
(``selective_scan``) and adds the result to the residual stream.  All tensors
are time-major, as ``RolloutBuffer`` stores them: ``[T, N, ...]`` for T steps
of N envs.  ``resets`` (bool or uint8 ``[T, N]``) is set where an env begins an
episode at that step: nothing from before reaches it, whatever it holds, so
episodes of any length lie one after the other in a row.

The whole-rollout forms are differentiable, once and in reverse (the learner); a
tangent of forward mode raises ``NotImplementedError``.  The carried state is
not differentiable: gradients stop where a rollout begins.  ``*_step`` is the
actor's form, one step of every env with the state updated in place.

Inputs are CUDA tensors of float32, bfloat16 or float16 whose last dimension
is contiguous (others are copied); other dimensions may have any stride, so
parts of a projection's output go in as they are.  Parameters (weights, rates,
biases) may be of any floating-point type and are taken in 32 bits.  States,
step sizes, sums and statistics are held in 32 bits; every output is rounded
once.  Calls enqueue on torch's current stream of the tensors' device and never
synchronise.  Bad arguments raise ``ValueError`` (``TypeError`` for what is no
tensor); there is no fallback without the library.
"""

from __future__ import annotations

from .._torch_ops import ext

FP8_GROUP = 128  # channels that share a scale


def _silu(activation: str | None) -> bool:
    if activation not in ("silu", None):
        raise ValueError(f"activation must be 'silu' or None, got {activation!r}")
    return activation == "silu"


def rms_norm(x, weight, residual=None, *, eps: float = 1e-6):
    """``s * rsqrt(mean(s**2) + eps) * weight`` over the last dimension.

    Without ``residual``, s is ``x`` and the result is one tensor.  With it, s
    is ``x + residual`` rounded to their type, and the result is ``(y, s)``: s
    is the residual stream that the next block adds to.  Differentiable in x,
    weight and residual."""
    out = ext.rms_norm(x, weight, residual, eps)
    return out[0] if residual is None else tuple(out)


def rms_norm_fp8(x, weight, residual=None, *, eps: float = 1e-6, group: int | None = None):
    """``rms_norm`` with y in 8 bits: ``(q, scale)`` or ``(q, scale, s)``.

    q is ``torch.float8_e4m3fn`` and stands for ``q * scale``.  ``group=None``:
    one scale a row (``scale`` has x's shape without the last dimension), as
    row-scaled matrix products take it; ``group=128``: one for each 128 channels
    (``[..., ceil(D / 128)]``).  A scale is the largest absolute value of its
    channels (at least 1e-30) divided by 448, so no value saturates.  Serving
    only: no gradient."""
    if group not in (None, FP8_GROUP):
        raise ValueError(f"group must be None or {FP8_GROUP}, got {group}")
    return tuple(ext.rms_norm_fp8(x, weight, residual, eps, group or 0))


def causal_conv(x, weight, bias=None, *, state=None, resets=None, activation: str | None = "silu"):
    """Convolution of each channel with its last ``width`` steps.

    ``x`` ``[T, N, D]``, ``weight`` ``[D, width]`` with width 2 to 4 (the last
    column weighs the current step), ``bias`` ``[D]``.  ``state``
    ``[N, width - 1, D]`` of x's type holds the inputs before the first step,
    oldest first (None: zeros).  Returns ``(y, state after the last step)``;
    differentiable in x, weight and bias."""
    return tuple(ext.causal_conv(x, weight, bias, state, resets, _silu(activation)))


def causal_conv_step(x, weight, bias, state, *, resets=None, activation: str | None = "silu"):
    """One step of ``causal_conv``: ``x`` ``[N, D]`` -> y ``[N, D]``; ``state``
    ``[N, width - 1, D]`` is moved on in place (where ``resets`` ``[N]`` is set,
    from zeros).  No gradient."""
    return ext.causal_conv_step(x, weight, bias, state, resets, _silu(activation))


def selective_scan(x, dt, A, B, C, D=None, z=None, *, dt_bias=None, softplus: bool = True, state=None, resets=None):
    """Selective state space recurrence along the steps.

    With ``delta = softplus(dt + dt_bias)`` (``softplus=False``: as it is)::

        h = exp(delta * A) * h + delta * B * x        (h = 0 before a step where an episode begins)
        y = (C . h + D * x) * silu(z)

    ``x``, ``dt``, ``z`` ``[T, N, channels]``; ``A`` ``[channels, states]``, up
    to 32 states; ``B``, ``C`` ``[T, N, groups, states]`` or ``[T, N, states]``,
    each group shared by ``channels / groups`` neighbouring channels; ``D``,
    ``dt_bias`` ``[channels]``; D, z and dt_bias may be None.  ``state``
    ``[N, channels, states]`` float32 before the first step (None: zeros).
    Returns ``(y, state after the last step)``; differentiable in everything
    but the state.  For the gradient every 8th state is kept."""
    return tuple(ext.selective_scan(x, dt, A, B, C, D, z, dt_bias, softplus, state, resets))


def selective_scan_step(x, dt, A, B, C, D=None, z=None, *, state, dt_bias=None, softplus: bool = True, resets=None):
    """One step of ``selective_scan``: ``x``, ``dt``, ``z`` ``[N, channels]``,
    ``B``, ``C`` ``[N, groups, states]`` or ``[N, states]`` -> y
    ``[N, channels]``; ``state`` ``[N, channels, states]`` float32 is updated in
    place (where ``resets`` ``[N]`` is set, from zeros).  No gradient."""
    return ext.selective_scan_step(x, dt, A, B, C, D, z, state, dt_bias, softplus, resets)
