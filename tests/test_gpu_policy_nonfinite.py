"""Values that are not finite, or would not be, where nothing may come from them."""

from __future__ import annotations

import pytest
import torch

from . import _policy_ref as ref
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


@pytest.mark.parametrize("states", [8, 12, 20])
def test_scan_gradient_of_an_infinite_step_size_that_is_left_out(states):
    """One channel forgets everything in a step of infinite size, as it does in
    one of size 300 (e^-300 is zero in 32 bits); that step is left out of the
    loss and an episode begins after it.  33 channels leave lanes of the kernel
    without one, 12 and 20 states without a state."""
    case = (24, 2, 33, states, 1, F32, 0.0, True, True, True, True, True)
    gen, t, state, _ = _scan_inputs(case)
    t["A"] = -1.0 - torch.rand(33, states, device="cuda", generator=gen)
    resets = torch.zeros(24, 2, dtype=torch.bool, device="cuda")
    resets[12, 0] = True
    dy = _randn(gen, 24, 2, 33)
    dy[11, 0] = 0
    got = {}
    for size in (300.0, float("inf")):
        t["dt"] = t["dt"].clone()
        t["dt"][11, 0, 32] = size
        got[size] = _gradients(t, dy, state, resets)
    fine = torch.ones(24, 2, dtype=torch.bool, device="cuda")
    fine[11, 0] = False
    for k in ("x", "dt", "B", "C", "z"):
        assert torch.isfinite(got[300.0][k]).all()
        assert torch.equal(got[float("inf")][k][fine], got[300.0][k][fine]), k
    assert torch.equal(got[float("inf")]["A"][:32], got[300.0]["A"][:32])


@pytest.mark.parametrize("steps", [64, 300, 1100])  # 4, 19 and 69 pieces: joined by the pass itself, in a row and in runs
def test_growth_of_nothing_is_nothing(steps):
    """States that grow by e^8 a step hold nothing until the last two steps
    push: over 16 steps the growth alone is e^128, beyond 32 bits.  The same
    against the steps for the gradient, where only the first two count."""
    from gbxcule_amd.rl import selective_scan

    gen = _gen(steps)
    x, b, c = _randn(gen, steps, 1, 40), _randn(gen, steps, 1, 16), _randn(gen, steps, 1, 16)
    x[:-2] = 0
    dt = torch.ones_like(x)
    rate = torch.full((40, 16), 8.0, device="cuda")
    dy = _randn(gen, steps, 1, 40)
    dy[2:] = 0
    x, dt, rate, b, c = _leaf(x, dt, rate, b, c)
    y, last = selective_scan(x, dt, rate, b, c, softplus=False)
    wide = [ref.f64(v) for v in (x, dt, rate, b.unsqueeze(2), c.unsqueeze(2))]
    want, want_last = ref.selective_scan(*wide, None, None, None, False, None, None)
    ref.check(y, want, 128, "y")
    ref.check(last, want_last, 128, "state")
    got = torch.autograd.grad(y, (x, dt, rate, b, c), dy)
    exact = torch.autograd.grad(want, wide, ref.f64(dy))
    for g, v, name in zip(got, exact, ("x", "dt", "A", "B", "C")):
        ref.check(g, v.view(g.shape), 256, f"gradient of {name}")
