"""The policy operators and autograd: what has no derivative, what is refused, and what a refusal leaves as it was."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from .conftest import require_gpu
from .test_gpu_policy_ops import _gen, _randn

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
