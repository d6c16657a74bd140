"""The policy operators and autograd: what has no derivative, what is refused, and what a refusal leaves as it was."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from .conftest import require_gpu
from .test_gpu_policy_ops import BF16, F32, _gen, _leaf, _randn

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu():
    require_gpu()


def _calls():
    """Name, function, its tensors."""
    from gbxcule_amd.rl import causal_conv, causal_conv_step, rms_norm, rms_norm_fp8, selective_scan, selective_scan_step

    g = _gen(1)
    x, w, r = _randn(g, 5, 3, 16), _randn(g, 16), _randn(g, 5, 3, 16)
    cw, window, h = _randn(g, 16, 4), _randn(g, 3, 3, 16), _randn(g, 3, 16, 8)
    dt, A, bc = _randn(g, 5, 3, 16), -torch.rand(16, 8, device="cuda", generator=g), _randn(g, 5, 3, 8)
    return [
        ("rms_norm", rms_norm, (x, w, r)),
        ("rms_norm_fp8", rms_norm_fp8, (x, w, r)),
        ("causal_conv", lambda x, w, b, s: causal_conv(x, w, b, state=s), (x, cw, w, window)),
        ("causal_conv_step", causal_conv_step, (x[0].clone(), cw, w, window)),
        ("selective_scan", lambda *a: selective_scan(*a[:7], dt_bias=a[7], state=a[8]), (x, dt, A, bc, bc.clone(), w, r, w.clone(), h)),
        ("selective_scan_step", lambda *a: selective_scan_step(*a[:7], dt_bias=a[7], state=a[8]),
         (x[0].clone(), dt[0].clone(), A, bc[0].clone(), bc[1].clone(), w, r[0].clone(), w.clone(), h)),
    ]  # fmt: skip


@pytest.mark.parametrize("which", range(6))
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(which, grad):
    """A tangent on any one argument: no output without one, and no state moved."""
    name, call, tensors = _calls()[which]
    for k, t in enumerate(tensors):
        kept = tensors[-1].clone()
        with torch.set_grad_enabled(grad), forward_ad.dual_level():
            dual = forward_ad.make_dual(t, torch.ones_like(t))
            with pytest.raises(NotImplementedError, match="forward"):
                call(*tensors[:k], dual, *tensors[k + 1 :])
        assert torch.equal(tensors[-1], kept), (name, k)
    call(*tensors)


def test_no_second_derivative():
    for name, call, tensors in _calls():
        if name not in ("rms_norm", "causal_conv", "selective_scan"):
            continue
        x = tensors[0].clone().requires_grad_()
        out = call(x, *tensors[1:])
        (g,) = torch.autograd.grad(out[0].sum(), x, retain_graph=True)
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(out[0].sum(), x, create_graph=True)
        assert torch.equal(g, torch.autograd.grad(out[0].sum(), x)[0])


def test_a_state_that_may_not_be_changed_is_not():
    """torch refuses to change an inference tensor outside inference mode."""
    for name, call, tensors in _calls():
        if not name.endswith("_step"):
            continue
        with torch.inference_mode():
            state = tensors[-1].clone()
            kept = state.clone()
        with torch.no_grad(), pytest.raises(RuntimeError, match="inference"):
            call(*tensors[:-1], state)
        torch.cuda.synchronize()
        assert torch.equal(state, kept), name
        with torch.inference_mode():
            y = call(*tensors[:-1], state)
        mine = tensors[-1].clone()
        version = mine._version
        assert torch.equal(call(*tensors[:-1], mine), y) and torch.equal(mine, state) and mine._version > version, name


@pytest.mark.parametrize("steps, envs", [(0, 3), (4, 0), (0, 0)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_empty_rollouts_keep_their_graph(steps, envs, dtype):
    """As with torch's operators: gradients of the inputs' shapes, zero for parameters."""
    from gbxcule_amd.rl import causal_conv, rms_norm, selective_scan

    g = _gen(2)
    rows = lambda d: _randn(g, steps, envs, d, dtype=dtype)  # noqa: E731
    resets = torch.zeros(steps, envs, dtype=torch.bool, device="cuda")
    window, h = _randn(g, envs, 3, 16, dtype=dtype), _randn(g, envs, 16, 8)
    norm = _leaf(rows(16), _randn(g, 16), rows(16))
    conv = _leaf(rows(16), _randn(g, 16, 4, dtype=BF16), _randn(g, 16))
    scan = _leaf(rows(16), rows(16), _randn(g, 16, 8), rows(8), rows(8), _randn(g, 16), rows(16), _randn(g, 16))
    for state in (True, False):
        results = [
            (norm, rms_norm(*norm)[0]),
            (conv, *causal_conv(*conv, state=window if state else None, resets=resets)),
            (scan, *selective_scan(*scan[:7], dt_bias=scan[7], state=h if state else None, resets=resets)),
        ]
        for (leaves, y, *last), kept in zip(results, (None, window, h)):
            assert y.shape == (steps, envs, 16) and y.dtype is dtype and y.requires_grad
            if last:
                assert last[0].shape == kept.shape and last[0].dtype is kept.dtype and not last[0].requires_grad
                assert torch.equal(last[0], kept if state else torch.zeros_like(kept)) and (envs == 0 or last[0].data_ptr() != kept.data_ptr())
            for v, t in zip(torch.autograd.grad(y, leaves, torch.ones_like(y)), leaves):
                assert v.shape == t.shape and v.dtype is t.dtype and not v.any()
    # a parameter alone wants a gradient
    for k in (2, 5, 7):
        one = [t.detach() for t in scan]
        one[k].requires_grad_()
        selective_scan(*one[:7], dt_bias=one[7])[0].sum().backward()
        assert one[k].grad is not None and not one[k].grad.any()
