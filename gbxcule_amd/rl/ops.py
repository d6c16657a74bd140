"""Operators of a policy that remembers an episode, as HIP kernels.

A memory block normalises its input (``rms_norm``, ``layer_norm``), mixes the
last few steps of each env (``causal_conv``), carries a state along the steps
(``selective_scan``, or a matrix a head: ``delta_rule``) and adds the result to
the residual stream; an actor draws from the logits that come out
(``sample_actions``).  All tensors are time-major, as ``RolloutBuffer`` stores them: ``[T, N, ...]`` for T steps
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


def layer_norm(x, weight, bias=None, residual=None, *, eps: float = 1e-5):
    """``(s - mean(s)) * rsqrt(mean((s - mean(s))**2) + eps) * weight + bias``
    over the last dimension; ``bias`` may be None.

    s, ``residual`` and the result are as in ``rms_norm``: y, or ``(y, s)``.
    Differentiable in x, weight, bias and residual."""
    out = ext.layer_norm(x, weight, bias, residual, eps)
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


def delta_rule(q, k, v, g, beta, *, scale: float | None = None, normalize: bool = True, state=None, resets=None):
    """Gated delta rule along the steps: a matrix S for each head, corrected
    towards what its key should recall::

        S = exp(g) * S                          (S = 0 before a step where an episode begins)
        S = S + k (beta * (v - S^T k))^T
        y = scale * S^T q

    ``q``, ``k`` ``[T, N, heads / share, keys]``, each of their heads shared by
    ``share`` neighbouring heads of ``v`` ``[T, N, heads, values]``; up to 128
    keys and values.  ``g`` (the logarithm of the decay, mostly below 0; below
    -104 it clears the state as an episode's start does) and ``beta`` ``[T, N,
    heads]`` are taken in 32 bits.  ``normalize``: q and k are divided by
    ``sqrt(sum of squares + 1e-6)``.  ``scale=None``: ``keys ** -0.5``.
    ``state`` ``[N, heads, keys, values]`` float32 before the first step (None:
    zeros).  Returns ``(y, state after the last step)``; differentiable in
    everything but the state.  For the gradient every 16th state is kept, and
    a value's correction at every step."""
    return tuple(ext.delta_rule(q, k, v, g, beta, scale, normalize, state, resets))


def delta_rule_step(q, k, v, g, beta, *, state, scale: float | None = None, normalize: bool = True, resets=None):
    """One step of ``delta_rule``: ``q``, ``k`` ``[N, heads / share, keys]``,
    ``v`` ``[N, heads, values]``, ``g``, ``beta`` ``[N, heads]`` -> y ``[N, heads,
    values]``; ``state`` ``[N, heads, keys, values]`` float32 is updated in place
    (where ``resets`` ``[N]`` is set, from zeros).  No gradient."""
    return ext.delta_rule_step(q, k, v, g, beta, state, scale, normalize, resets)


def sample_actions(logits, uniform, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Actions drawn from ``logits`` ``[..., actions]`` with the random numbers
    ``uniform`` ``[...]`` (float32, from 0 to below 1): ``(action int32 [...],
    logp float32 [...])``.

    Weights are ``exp(logits / temperature)``; temperature 0 takes the largest
    logit.  From the likeliest action on, the lowest index first among equals, a
    row keeps its first ``top_k`` (0: all), of those the fewest that hold
    ``top_p`` of their weight (1: all), of those all with at least ``min_p`` of the
    largest weight, and always one.  ``action`` is the first index at which the
    running sum of the kept weights passes ``uniform`` times their sum, and
    ``logp`` the logarithm of the probability it was drawn with.  Each option is a
    number or a tensor ``[...]`` with one for each row (float32, ``top_k`` int32).

    NaN and -infinity are never drawn; a row of nothing else has action -1 and
    logp NaN.  Weights and sums are in 64 bits.  No gradient, of the logits or
    the options."""
    return tuple(ext.sample_actions(logits, uniform, temperature, top_k, top_p, min_p))
