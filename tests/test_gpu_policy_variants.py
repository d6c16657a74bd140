"""Policy operators at sizes where a workgroup takes more than one turn, where
the single steps take several envs a lane, and from several threads at once."""

from __future__ import annotations

import threading

import pytest
import torch

from . import _policy_ref as ref
from .conftest import require_gpu
from .test_gpu_policy_ops import BF16, F16, F32, NAMES, _gen, _leaf, _randn, _scan_inputs

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu():
    require_gpu()


# rows beyond those of 1,024 workgroups, in each shape of the kernel's rows
@pytest.mark.parametrize("rows, dim, dtype", [(17_000, 100, F32), (9_000, 256, BF16), (5_000, 1_000, F32), (5_000, 513, F16), (1_100, 2_049, F32),
                                              (1_100, 4_096, BF16), (1_030, 8_191, F32), (1_100, 8_200, F32), (2_060, 9_001, BF16), (17_000, 7, F32)])  # fmt: skip
def test_norm_gradient_of_many_rows(rows, dim, dtype):
    from gbxcule_amd.rl import rms_norm

    gen = _gen(rows + dim)
    x, w, r = _randn(gen, rows, dim, dtype=dtype), 1.0 + _randn(gen, dim, scale=0.2), _randn(gen, rows, dim, dtype=dtype)
    dy, ds = _randn(gen, rows, dim, dtype=dtype), _randn(gen, rows, dim, dtype=dtype)
    leaves = _leaf(x, w, r)
    out = rms_norm(*leaves, eps=1e-5)
    got = torch.autograd.grad(out, leaves, [dy, ds], retain_graph=True)
    again = torch.autograd.grad(out, leaves, [dy, ds])
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    # the formula: with g = w dy and inv = 1 / root, ds = inv g - s inv^3 mean(g s) + ds_out, dw = sum dy s inv
    s, dyw, wide_w = out[1].detach().cpu().double(), dy.cpu().double(), w.cpu().double()
    assert torch.equal(out[1].detach().cpu(), (x.float() + r.float()).to(dtype).cpu())
    inv = 1.0 / torch.sqrt((s * s).mean(-1, keepdim=True) + 1e-5)
    pull = (wide_w * dyw * s).mean(-1, keepdim=True)
    dx = inv * wide_w * dyw - s * inv**3 * pull + ds.cpu().double()
    # a row's sums go through the lanes' own adds and the tree between them; the weight's gradient through a
    # workgroup's turns, then 1,024 / 64 partial sums in a row and a tree of 64
    n = 16 + 3 * dim.bit_length() + dim // 256
    ref.check(out[0], s * inv * wide_w, n, "y")
    ref.check(got[0], dx, 2 * n, "gradient of x")
    assert torch.equal(got[0], got[2])
    ref.check(got[1], (dyw * s * inv).sum(0), 2 * n + rows // 1024 + 32, "gradient of weight")


@pytest.mark.parametrize("case", [
    # (env, piece) items beyond the workgroups that the gradient has for them
    (2, 5000, 33, 16, 1, F32, 0.3, True, True, True, True, True),
    (64, 600, 33, 16, 1, F32, 0.05, True, True, True, True, True),  # cut along the steps
    (9, 700, 200, 16, 1, BF16, 0.1, True, True, True, True, True),  # two channel blocks to a group
    (3, 2500, 72, 8, 2, F32, 0.3, True, False, True, True, True),
    (11, 1200, 40, 32, 1, F32, 0.1, False, True, True, True, True),
    (9, 1100, 40, 24, 1, F16, 0.0, True, True, False, False, False),
], ids=str)  # fmt: skip
def test_scan_gradient_of_many_rows(case):
    from gbxcule_amd.rl import selective_scan

    steps, envs, dim, states, groups, dtype, softplus = *case[:6], case[10]
    gen, t, state, resets = _scan_inputs(case)
    leaf = dict(zip(NAMES, _leaf(*(t[k] for k in NAMES))))
    y, last = selective_scan(*(leaf[k] for k in NAMES[:7]), dt_bias=leaf["dt_bias"], softplus=softplus, state=state, resets=resets)
    wide = {k: ref.f64(leaf[k]) for k in NAMES}
    want, want_last = ref.selective_scan(*(wide[k] for k in NAMES), softplus, ref.f64(state), None if resets is None else resets.cpu())
    n = 128 + steps
    ref.check(y, want, n, "y")
    ref.check(last, want_last, n, "state")
    dy = _randn(gen, steps, envs, dim, dtype=dtype)
    names = [k for k in NAMES if leaf[k] is not None]
    got = torch.autograd.grad(y, [leaf[k] for k in names], dy, retain_graph=True)
    again = torch.autograd.grad(y, [leaf[k] for k in names], dy)
    exact = torch.autograd.grad(want, [wide[k] for k in names], ref.f64(dy))
    for g, a, v, name in zip(got, again, exact, names):
        assert torch.equal(g, a), name  # no order that changes
        # parameters: a workgroup's turns (up to 3 of 16 steps) and 2,048 / 64 partial sums in a row, a tree of 64
        ref.check(g, v, 2 * n + (128 if name in ("A", "D", "dt_bias") else dim), f"gradient of {name}")


@pytest.mark.parametrize("dim, width, dtype", [(512, 4, BF16), (509, 4, BF16), (509, 3, F32), (512, 2, F16), (507, 2, F32)])
def test_conv_step_of_many_envs(dim, width, dtype):
    """From 524,288 lanes on a lane takes four envs: the same as in parts that are smaller."""
    from gbxcule_amd.rl import causal_conv_step

    gen, envs = _gen(dim + width), 20_011
    assert envs * -(-dim // 8) >= 524_288
    x, w, b = _randn(gen, envs, dim, dtype=dtype), _randn(gen, dim, width, scale=0.5), _randn(gen, dim)
    state = _randn(gen, envs, width - 1, dim, dtype=dtype)
    resets = torch.rand(envs, device="cuda", generator=gen) < 0.2
    small, parts = state.clone(), 5_003
    assert parts * -(-dim // 8) < 524_288
    y = causal_conv_step(x, w, b, state, resets=resets)
    for at in range(0, envs, parts):
        to = slice(at, at + parts)
        assert torch.equal(y[to], causal_conv_step(x[to], w, b, small[to], resets=resets[to])), at
    assert torch.equal(state, small)
    assert torch.equal(state[:, -1], x)


@pytest.mark.parametrize("states, dtype, groups", [(4, F32, 1), (8, BF16, 2), (12, F32, 1), (16, F16, 1), (20, BF16, 4), (24, F32, 1), (28, F32, 2), (32, BF16, 1)])
def test_scan_step_of_many_envs(states, dtype, groups):
    from gbxcule_amd.rl import selective_scan_step

    envs, dim, parts = 10_007, 64, 701
    _, t, state, _ = _scan_inputs((1, envs, dim, states, groups, dtype, 0.0, True, True, True, True, True))
    gen = _gen(states)
    resets = torch.rand(envs, device="cuda", generator=gen) < 0.2
    row = {k: v[0] if k in ("x", "dt", "B", "C", "z") else v for k, v in t.items()}
    small = state.clone()

    def step(part, h):
        cut = [row[k][part] if k in ("x", "dt", "B", "C", "z") else row[k] for k in NAMES[:7]]
        return selective_scan_step(*cut, state=h, dt_bias=row["dt_bias"], resets=resets[part])

    y = step(slice(None), state)
    for at in range(0, envs, parts):
        part = slice(at, at + parts)
        assert torch.equal(y[part], step(part, small[part])), at
    assert torch.equal(state, small) and torch.isfinite(state).all()


def test_threads_with_streams_of_their_own():
    """Calls release the interpreter: four threads, forward and backward."""
    from gbxcule_amd.rl import causal_conv, rms_norm, selective_scan

    inputs = [_scan_inputs((40, 3, 64, 16, 1, F32, 0.1, True, True, True, True, True)) for _ in range(4)]
    weights = [(_randn(_gen(k), 64, 4), 1 + _randn(_gen(9 + k), 64, scale=0.1)) for k in range(4)]
    for k, (gen, t, _, _) in enumerate(inputs):
        t["x"] = _randn(_gen(50 + k), 40, 3, 64)

    def work(k):
        _, t, state, resets = inputs[k]
        leaf = dict(zip(NAMES, _leaf(*(None if t[n] is None else t[n].clone() for n in NAMES))))
        cw, nw = _leaf(*(w.clone() for w in weights[k]))
        u, _ = causal_conv(rms_norm(leaf["x"], nw), cw, resets=resets)
        y, last = selective_scan(u, *(leaf[n] for n in NAMES[1:7]), dt_bias=leaf["dt_bias"], state=state, resets=resets)
        return [y.detach(), last, *torch.autograd.grad(y.square().sum(), [leaf["x"], leaf["A"], leaf["B"], cw, nw])]

    want = [work(k) for k in range(4)]
    torch.cuda.synchronize()
    got: list = [None] * 4

    def run(k):
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            for _ in range(10):
                got[k] = work(k)
        side.synchronize()

    threads = [threading.Thread(target=run, args=(k,)) for k in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    for a, b in zip(got, want):
        assert a is not None and all(torch.equal(u, v) for u, v in zip(a, b))
