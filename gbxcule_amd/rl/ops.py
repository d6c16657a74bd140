"""Operators of a policy that remembers an episode, as HIP kernels.

A memory block normalises its input (``rms_norm``), mixes the last few steps
of each env (``causal_conv``), carries a state along the steps
(``selective_scan``) and adds the result to the residual stream.  All tensors
are time-major, as ``RolloutBuffer`` stores them: ``[T, N, ...]`` for T steps
of N envs.  ``resets`` (bool or uint8 ``[T, N]``) is set where an env begins an
episode at that step: nothing from before reaches it, whatever it holds, so
episodes of any length lie one after the other in a row.

The whole-rollout forms are differentiable (the learner); the carried state is
not: gradients stop where a rollout begins.  ``*_step`` is the actor's form,
one step of every env with the state updated in place.

Inputs are CUDA tensors of float32, bfloat16 or float16 whose last dimension
is contiguous (others are copied); other dimensions may have any stride, so
parts of a projection's output go in as they are.  States, step sizes, sums
and statistics are held in 32 bits; every output is rounded once.  Calls
enqueue on torch's current stream of the tensors' device and never
synchronise.  There is no fallback: without the library every call raises.
"""

from __future__ import annotations

from typing import Any

import torch

from .. import _lib

_ELEM = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
FP8_GROUP = 128  # channels that share a scale


def _require(ok: bool, message: str) -> None:
    if not ok:
        raise ValueError(message)


def _elem(name: str, t: torch.Tensor) -> int:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor, got one on {t.device}")
    elem = _ELEM.get(t.dtype)
    if elem is None:
        raise ValueError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    return elem


def _like(name: str, t: torch.Tensor, like: torch.Tensor, shape: tuple[int, ...]) -> torch.Tensor:
    """``t`` of ``like``'s type and device and the given shape, last dimension contiguous."""
    if t.dtype is not like.dtype or t.get_device() != like.get_device():
        raise ValueError(f"{name}: expected {like.dtype} on {like.device}, got {t.dtype} on {t.device}")
    if t.shape != shape:
        raise ValueError(f"{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    return _rows(t)


def _rows(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _param(name: str, t: torch.Tensor | None, like: torch.Tensor, shape: tuple[int, ...]) -> torch.Tensor | None:
    """A parameter in 32 bits (the cast is differentiable), contiguous."""
    if t is None:
        return None
    if t.get_device() != like.get_device() or not t.is_floating_point():
        raise ValueError(f"{name}: expected a floating-point tensor on {like.device}, got {t.dtype} on {t.device}")
    if t.shape != shape:
        raise ValueError(f"{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.dtype is not torch.float32:
        t = t.float()
    return t if t.is_contiguous() else t.contiguous()


def _resets(t: torch.Tensor | None, like: torch.Tensor, shape: tuple[int, ...]) -> torch.Tensor | None:
    if t is None:
        return None
    if t.dtype not in (torch.bool, torch.uint8) or t.get_device() != like.get_device():
        raise ValueError(f"resets: expected bool or uint8 on {like.device}, got {t.dtype} on {t.device}")
    if t.shape != shape:
        raise ValueError(f"resets: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    return t.contiguous()


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _call(fn: str, t: torch.Tensor, *args: Any) -> None:
    """A launch on the current stream of ``t``'s device.  (The raw stream
    getter: a ``torch.cuda.Stream`` object costs as much as the launch.)"""
    device = t.get_device()
    entry = getattr(_lib.load(), fn)
    if device == torch.cuda.current_device():
        rc = entry(*args, torch._C._cuda_getCurrentRawStream(device))
    else:
        with torch.cuda.device(device):
            rc = entry(*args, torch._C._cuda_getCurrentRawStream(device))
    if rc:
        _lib.check(rc)


def _empty_like(t: torch.Tensor) -> torch.Tensor:
    """Contiguous, of t's shape, type and device."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _work(count: int, like: torch.Tensor) -> torch.Tensor | None:
    if count < 0:
        _lib.check(int(count))
    return torch.empty(count, dtype=torch.float32, device=like.device) if count else None


def _wants_grad(*tensors: torch.Tensor | None) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _no_grad(what: str, *tensors: torch.Tensor | None) -> None:
    if _wants_grad(*tensors):
        raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad() or with detached tensors")


# ------------------------------------------------------------------ the norm


def _flat(t: torch.Tensor) -> torch.Tensor:
    """``[..., D]`` as rows ``[R, D]`` with a contiguous last dimension."""
    t = _rows(t)
    return t if t.ndim == 2 else t.reshape(-1, t.shape[-1])


def _norm_operands(x, weight, residual):
    elem = _elem("x", x)
    _require(x.ndim >= 1 and x.shape[-1] >= 1, f"x: expected [..., channels], got {tuple(x.shape)}")
    weight = _param("weight", weight, x, (x.shape[-1],))
    if residual is not None:
        residual = _like("residual", residual, x, x.shape)
    return elem, weight, residual


def _norm_forward(elem, x, weight, residual, eps, out, scale=None, group=0):
    rows, dim = _flat(x), x.shape[-1]
    res = None if residual is None else _flat(residual)
    summed = None if res is None else _empty_like(x)
    _call("gbx_rms_norm", x, rows.shape[0], dim, elem, eps, rows.data_ptr(), rows.stride(0), _ptr(res),
          0 if res is None else res.stride(0), weight.data_ptr(), out.data_ptr(), _ptr(summed), _ptr(scale), group)  # fmt: skip
    return summed


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps, elem):
        ctx.set_materialize_grads(False)
        y = _empty_like(x)
        summed = _norm_forward(elem, x, weight, residual, eps, y)
        ctx.save_for_backward(x if residual is None else summed, weight)
        ctx.eps, ctx.elem, ctx.plain = eps, elem, residual is None
        return y if residual is None else (y, summed)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dsummed=None):
        s, weight = ctx.saved_tensors
        dim = s.shape[-1]
        if dy is None or s.numel() == 0:  # the sum alone was used, or there are no rows
            dx = torch.zeros_like(s) if dsummed is None else dsummed
            return dx, torch.zeros_like(weight), None if ctx.plain else dx, None, None
        rows, dy = _flat(s), _flat(dy)
        if dsummed is not None:
            dsummed = _flat(dsummed)
        dx = _empty_like(s)
        dweight = torch.empty_like(weight)
        work = _work(_lib.load().gbx_rms_norm_grad_work(rows.shape[0], dim), s)
        _call("gbx_rms_norm_grad", s, rows.shape[0], dim, ctx.elem, ctx.eps, rows.data_ptr(), rows.stride(0),
              dy.data_ptr(), dy.stride(0), _ptr(dsummed), 0 if dsummed is None else dsummed.stride(0),
              weight.data_ptr(), dx.data_ptr(), dweight.data_ptr(), work.data_ptr())  # fmt: skip
        return dx, dweight, None if ctx.plain else dx, None, None


def rms_norm(x, weight, residual=None, *, eps: float = 1e-6):
    """``s * rsqrt(mean(s**2) + eps) * weight`` over the last dimension.

    Without ``residual``, s is ``x`` and the result is one tensor.  With it, s
    is ``x + residual`` rounded to their type, and the result is ``(y, s)``: s
    is the residual stream that the next block adds to.  Differentiable in x,
    weight and residual."""
    elem, weight, residual = _norm_operands(x, weight, residual)
    if _wants_grad(x, weight, residual):
        return _RmsNorm.apply(x, weight, residual, float(eps), elem)
    y = _empty_like(x)
    summed = _norm_forward(elem, x, weight, residual, float(eps), y) if x.numel() else y
    return y if residual is None else (y, summed)


def rms_norm_fp8(x, weight, residual=None, *, eps: float = 1e-6, group: int | None = None):
    """``rms_norm`` with y in 8 bits: ``(q, scale)`` or ``(q, scale, s)``.

    q is ``torch.float8_e4m3fn`` and stands for ``q * scale``.  ``group=None``:
    one scale a row (``scale`` has x's shape without the last dimension), as
    row-scaled matrix products take it; ``group=128``: one for each 128 channels
    (``[..., ceil(D / 128)]``).  A scale is the largest absolute value of its
    channels (at least 1e-30) divided by 448, so no value saturates.  Serving
    only: no gradient."""
    _no_grad("rms_norm_fp8", x, weight, residual)
    _require(group in (None, FP8_GROUP), f"group must be None or {FP8_GROUP}, got {group}")
    elem, weight, residual = _norm_operands(x, weight, residual)
    dim = x.shape[-1]
    q = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device)
    scales = x.shape[:-1] if group is None else (*x.shape[:-1], -(-dim // FP8_GROUP))
    scale = torch.empty(scales, dtype=torch.float32, device=x.device)
    if x.numel():
        summed = _norm_forward(elem, x, weight, residual, float(eps), q, scale, group or 0)
    else:
        summed = None if residual is None else torch.empty_like(x)
    return (q, scale) if residual is None else (q, scale, summed)


# ------------------------------------------------------- the causal convolution


def _silu(activation: str | None) -> int:
    _require(activation in ("silu", None), f"activation must be 'silu' or None, got {activation!r}")
    return int(activation == "silu")


def _conv_params(x, weight, bias):
    dim = x.shape[-1]
    _require(weight.ndim == 2 and 2 <= weight.shape[1] <= 4, f"weight: expected [channels, 2 to 4], got {tuple(weight.shape)}")
    return _param("weight", weight, x, (dim, weight.shape[1])), _param("bias", bias, x, (dim,))


def _conv_state(state, x, envs: int, width: int):
    if state is None:
        return None
    _require(not _wants_grad(state), "state carries no gradient: detach it")
    return _like("state", state, x, (envs, width - 1, x.shape[-1])).contiguous()


class _CausalConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state, resets, silu, elem):
        ctx.set_materialize_grads(False)
        steps, envs, dim = x.shape
        width = weight.shape[1]
        y = _empty_like(x)
        last = torch.empty((envs, width - 1, dim), dtype=x.dtype, device=x.device)
        _call("gbx_causal_conv", x, steps, envs, dim, width, elem, silu, x.data_ptr(), x.stride(0), x.stride(1),
              weight.data_ptr(), _ptr(bias), _ptr(state), _ptr(resets), y.data_ptr(), last.data_ptr())  # fmt: skip
        ctx.save_for_backward(x, weight, bias, state, resets)
        ctx.silu, ctx.elem = silu, elem
        ctx.mark_non_differentiable(last)
        return y, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, _):
        x, weight, bias, state, resets = ctx.saved_tensors
        if dy is None:
            return (None,) * 7
        steps, envs, dim = x.shape
        width = weight.shape[1]
        dy = _rows(dy)
        dx = _empty_like(x)
        dweight = torch.empty_like(weight)
        dbias = None if bias is None else torch.empty_like(bias)
        work = _work(_lib.load().gbx_causal_conv_grad_work(steps, envs, dim, width), x)
        _call("gbx_causal_conv_grad", x, steps, envs, dim, width, ctx.elem, ctx.silu, x.data_ptr(), x.stride(0),
              x.stride(1), weight.data_ptr(), _ptr(bias), _ptr(state), _ptr(resets), dy.data_ptr(), dy.stride(0),
              dy.stride(1), dx.data_ptr(), dweight.data_ptr(), _ptr(dbias), work.data_ptr())  # fmt: skip
        return dx, dweight, dbias, None, None, None, None


def causal_conv(x, weight, bias=None, *, state=None, resets=None, activation: str | None = "silu"):
    """Convolution of each channel with its last ``width`` steps.

    ``x`` ``[T, N, D]``, ``weight`` ``[D, width]`` with width 2 to 4 (the last
    column weighs the current step), ``bias`` ``[D]``.  ``state``
    ``[N, width - 1, D]`` of x's type holds the inputs before the first step,
    oldest first (None: zeros).  Returns ``(y, state after the last step)``;
    differentiable in x, weight and bias."""
    elem = _elem("x", x)
    _require(x.ndim == 3 and x.shape[2] >= 1, f"x: expected [steps, envs, channels], got {tuple(x.shape)}")
    x = _rows(x)
    weight, bias = _conv_params(x, weight, bias)
    steps, envs, dim = x.shape
    state = _conv_state(state, x, envs, weight.shape[1])
    resets = _resets(resets, x, (steps, envs))
    if x.numel() == 0:
        kept = (envs, weight.shape[1] - 1, dim)
        return x * weight.sum().to(x.dtype), x.new_zeros(kept) if state is None else state.clone()
    return _CausalConv.apply(x, weight, bias, state, resets, _silu(activation), elem)


def causal_conv_step(x, weight, bias, state, *, resets=None, activation: str | None = "silu"):
    """One step of ``causal_conv``: ``x`` ``[N, D]`` -> y ``[N, D]``; ``state``
    ``[N, width - 1, D]`` is moved on in place (where ``resets`` ``[N]`` is set,
    from zeros).  No gradient."""
    elem = _elem("x", x)
    _no_grad("causal_conv_step", x, weight, bias, state)
    _require(x.ndim == 2 and x.shape[1] >= 1, f"x: expected [envs, channels], got {tuple(x.shape)}")
    x = _rows(x)
    weight, bias = _conv_params(x, weight, bias)
    envs, dim = x.shape
    _like("state", state, x, (envs, weight.shape[1] - 1, dim))
    _require(state.is_contiguous(), "state must be contiguous: it is updated in place")
    resets = _resets(resets, x, (envs,))
    silu = _silu(activation)
    y = _empty_like(x)
    if envs:
        _call("gbx_causal_conv_step", x, envs, dim, weight.shape[1], elem, silu, x.data_ptr(), x.stride(0),
              weight.data_ptr(), _ptr(bias), state.data_ptr(), _ptr(resets), y.data_ptr())  # fmt: skip
        torch.autograd.graph.increment_version(state)
    return y


# ---------------------------------------------------------- the selective scan


def _scan_operands(x, dt, A, B, C, D, z, dt_bias, resets):
    """Checked operands; B and C with a group dimension."""
    dim, lead = x.shape[-1], x.shape[:-1]
    if B.ndim == x.ndim:
        B = B.unsqueeze(-2)
    if C.ndim == x.ndim:
        C = C.unsqueeze(-2)
    _require(A.ndim == 2 and 1 <= A.shape[1] <= 32, f"A: expected [channels, 1 to 32 states], got {tuple(A.shape)}")
    _require(B.ndim == x.ndim + 1 and B.shape[-2] >= 1 and dim % B.shape[-2] == 0,
             f"B: expected [..., groups, states] with groups dividing {dim}, got {tuple(B.shape)}")  # fmt: skip
    each = (*lead, B.shape[-2], A.shape[1])
    return (
        _like("dt", dt, x, x.shape), _param("A", A, x, (dim, A.shape[1])), _like("B", B, x, each),
        _like("C", C, x, each), _param("D", D, x, (dim,)), None if z is None else _like("z", z, x, x.shape),
        _param("dt_bias", dt_bias, x, (dim,)), _resets(resets, x, lead),
    )  # fmt: skip


def _scan_in(x, dt, A, B, C, D, z, dt_bias, resets, softplus, elem) -> _lib.ScanIn:
    one = x.ndim == 2  # a single step
    pair = lambda t: (0, t.stride(0)) if one else (t.stride(0), t.stride(1))  # noqa: E731
    return _lib.ScanIn(
        1 if one else x.shape[0], x.shape[-2], x.shape[-1], B.shape[-2], A.shape[1], elem, int(softplus),
        x.data_ptr(), dt.data_ptr(), _ptr(z), B.data_ptr(), C.data_ptr(),
        *pair(x), *pair(dt), *((0, 0) if z is None else pair(z)), *pair(B), B.stride(-2), *pair(C), C.stride(-2),
        A.data_ptr(), _ptr(D), _ptr(dt_bias), _ptr(resets),
    )  # fmt: skip


def _scan_forward(x, dt, A, B, C, D, z, dt_bias, state, resets, softplus, elem, save):
    steps, envs, dim = x.shape
    given = _scan_in(x, dt, A, B, C, D, z, dt_bias, resets, softplus, elem)
    y = _empty_like(x)
    last = torch.empty((envs, dim, A.shape[1]), dtype=torch.float32, device=x.device)
    saved = None
    if save:
        saved = torch.empty((-(-steps // 8), envs, dim, A.shape[1]), dtype=torch.float32, device=x.device)
    work = _work(_lib.load().gbx_selective_scan_work(given), x)
    _call("gbx_selective_scan", x, given, _ptr(state), y.data_ptr(), last.data_ptr(), _ptr(saved), _ptr(work))
    return y, last, saved


class _SelectiveScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, dt, A, B, C, D, z, dt_bias, state, resets, softplus, elem):
        ctx.set_materialize_grads(False)
        y, last, saved = _scan_forward(x, dt, A, B, C, D, z, dt_bias, state, resets, softplus, elem, True)
        ctx.save_for_backward(x, dt, A, B, C, D, z, dt_bias, resets, saved)
        ctx.softplus, ctx.elem = softplus, elem
        ctx.mark_non_differentiable(last)
        return y, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, _):
        x, dt, A, B, C, D, z, dt_bias, resets, saved = ctx.saved_tensors
        if dy is None:
            return (None,) * 12
        given = _scan_in(x, dt, A, B, C, D, z, dt_bias, resets, ctx.softplus, ctx.elem)
        dy = _rows(dy)
        dx, ddt, dA, dB, dC, dD, dz, dbias = (None if t is None else _empty_like(t) for t in (x, dt, A, B, C, D, z, dt_bias))
        work = _work(_lib.load().gbx_selective_scan_grad_work(given), x)
        _call("gbx_selective_scan_grad", x, given, saved.data_ptr(), dy.data_ptr(), dy.stride(0), dy.stride(1),
              dx.data_ptr(), ddt.data_ptr(), _ptr(dz), dB.data_ptr(), dC.data_ptr(), dA.data_ptr(), _ptr(dD),
              _ptr(dbias), work.data_ptr())  # fmt: skip
        return dx, ddt, dA, dB, dC, dD, dz, dbias, None, None, None, None


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
    elem = _elem("x", x)
    _require(x.ndim == 3 and x.shape[2] >= 1, f"x: expected [steps, envs, channels], got {tuple(x.shape)}")
    x = _rows(x)
    steps, envs, dim = x.shape
    dt, A, B, C, D, z, dt_bias, resets = _scan_operands(x, dt, A, B, C, D, z, dt_bias, resets)
    kept = (envs, dim, A.shape[1])
    if state is not None:
        _require(not _wants_grad(state), "state carries no gradient: detach it")
        state = _scan_state(state, x, kept).contiguous()
    if x.numel() == 0:
        last = torch.zeros(kept, dtype=torch.float32, device=x.device) if state is None else state.clone()
        return x * 0, last
    if _wants_grad(x, dt, A, B, C, D, z, dt_bias):
        return _SelectiveScan.apply(x, dt, A, B, C, D, z, dt_bias, state, resets, bool(softplus), elem)
    return _scan_forward(x, dt, A, B, C, D, z, dt_bias, state, resets, bool(softplus), elem, False)[:2]


def _scan_state(state, x, shape):
    if state.dtype is not torch.float32 or state.get_device() != x.get_device() or state.shape != shape:
        raise ValueError(f"state: expected float32 {shape} on {x.device}, got {state.dtype} {tuple(state.shape)} on {state.device}")
    return state


def selective_scan_step(x, dt, A, B, C, D=None, z=None, *, state, dt_bias=None, softplus: bool = True, resets=None):
    """One step of ``selective_scan``: ``x``, ``dt``, ``z`` ``[N, channels]``,
    ``B``, ``C`` ``[N, groups, states]`` or ``[N, states]`` -> y
    ``[N, channels]``; ``state`` ``[N, channels, states]`` float32 is updated in
    place (where ``resets`` ``[N]`` is set, from zeros).  No gradient."""
    elem = _elem("x", x)
    _no_grad("selective_scan_step", x, dt, A, B, C, D, z, dt_bias, state)
    _require(x.ndim == 2 and x.shape[1] >= 1, f"x: expected [envs, channels], got {tuple(x.shape)}")
    x = _rows(x)
    dt, A, B, C, D, z, dt_bias, resets = _scan_operands(x, dt, A, B, C, D, z, dt_bias, resets)
    _scan_state(state, x, (*x.shape, A.shape[1]))
    _require(state.is_contiguous(), "state must be contiguous: it is updated in place")
    y = _empty_like(x)
    if x.shape[0]:
        given = _scan_in(x, dt, A, B, C, D, z, dt_bias, resets, softplus, elem)
        _call("gbx_selective_scan_step", x, given, state.data_ptr(), y.data_ptr())
        torch.autograd.graph.increment_version(state)
    return y
