"""Values that are not finite, or would not be, where nothing may come from them."""

from __future__ import annotations

import pytest
import torch

from .conftest import require_gpu
from .test_gpu_policy_ops import BF16, F32, NAMES, _gen, _leaf, _randn, _scan_inputs

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu():
    require_gpu()


def _gradients(t, dy, state, resets, softplus=True):
    from gbxcule_amd.rl import selective_scan

    leaf = dict(zip(NAMES, _leaf(*(t[k] for k in NAMES))))
    y, _ = selective_scan(*(leaf[k] for k in NAMES[:7]), dt_bias=leaf["dt_bias"], softplus=softplus, state=state, resets=resets)
    names = [k for k in NAMES if leaf[k] is not None]
    return dict(zip(names, torch.autograd.grad(y, [leaf[k] for k in names], dy)))


@pytest.mark.parametrize("steps", [1, 13, 45, 203])  # none a multiple of the 8 steps that the gradient goes back at a time
@pytest.mark.parametrize("states, dtype", [(8, F32), (12, F32), (16, BF16), (32, F32)])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_scan_gradient_of_a_last_step_that_is_left_out(steps, states, dtype, bad):
    """The last step's input is not finite and the loss leaves its output out:
    what does not depend on that input is as if it were finite."""
    case = (steps, 2, 70, states, 1, dtype, 0.0, True, True, True, True, True)
    gen, t, state, resets = _scan_inputs(case)
    dy = _randn(gen, steps, 2, 70, dtype=dtype)
    dy[-1, 0] = 0
    want = _gradients(t, dy, state, resets)
    t["x"] = t["x"].clone()
    t["x"][-1, 0] = bad
    got = _gradients(t, dy, state, resets)
    fine = torch.ones(steps, 2, dtype=torch.bool, device="cuda")
    fine[-1, 0] = False
    assert torch.equal(got["A"], want["A"])  # the last state decays into nothing
    for k in ("x", "dt", "B", "C", "z"):
        assert torch.equal(got[k][fine], want[k][fine]), k
