"""Norm, causal convolution and selective scan against plain 64-bit forms:
sizes around every tile, types, strides, episode starts, values behind them
that must not be seen, gradients against autograd and against differences,
single steps against whole rollouts, and refusals."""

from __future__ import annotations

import pytest
import torch

from . import _policy_ref as ref
from .conftest import require_gpu

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _gpu():
    require_gpu()


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape, dtype=F32, scale=1.0):
    return (torch.randn(shape, device="cuda", generator=gen) * scale).to(dtype)


def _leaf(*tensors):
    return [None if t is None else t.detach().requires_grad_() for t in tensors]


# ------------------------------------------------------------------ the norm

# around the row lengths where the kernel's lanes and pieces change, odd ones
NORM_DIMS = [1, 7, 64, 127, 128, 129, 256, 257, 511, 512, 520, 1000, 1024, 1025, 2048, 2049, 4096, 4100, 8192, 8193, 20000]


@pytest.mark.parametrize("dim", NORM_DIMS)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("residual", [False, True])
def test_norm(dim, dtype, residual):
    from gbxcule_amd.rl import rms_norm

    gen = _gen(dim)
    rows = 5 if dim > 4000 else 37
    x, w = _randn(gen, rows, dim, dtype=dtype), 1.0 + _randn(gen, dim, scale=0.2)
    r = _randn(gen, rows, dim, dtype=dtype, scale=2.0) if residual else None
    dy, ds = _randn(gen, rows, dim, dtype=dtype), _randn(gen, rows, dim, dtype=dtype)
    leaves = [t for t in _leaf(x, w, r) if t is not None]
    out = rms_norm(leaves[0], leaves[1], leaves[2] if residual else None, eps=1e-5)
    wide = [ref.f64(t) for t in leaves]
    y, s = ref.rms_norm(wide[0], wide[1], wide[2] if residual else None, 1e-5, dtype)
    # a row's sum of squares goes through the lanes' own adds and the tree between them
    n = 16 + 3 * dim.bit_length() + dim // 256
    if residual:
        ref.check(out[0], y, n, "y")
        assert torch.equal(out[1].cpu().double(), s.detach())
        got = torch.autograd.grad(out, leaves, [dy, ds])
        want = torch.autograd.grad([y, s], wide, [ref.f64(dy), ref.f64(ds)])
        with torch.no_grad():
            again = rms_norm(x, w, r, eps=1e-5)
        assert torch.equal(again[0], out[0]) and torch.equal(again[1], out[1])
    else:
        ref.check(out, y, n, "y")
        got = torch.autograd.grad(out, leaves, dy)
        want = torch.autograd.grad(y, wide, ref.f64(dy))
    for g, v, name in zip(got, want, ("x", "weight", "residual")):
        ref.check(g, v, 2 * n + rows, f"gradient of {name}")


@pytest.mark.parametrize("dim", [1, 100, 128, 129, 512, 1000, 1024, 4096, 8192, 9000])
@pytest.mark.parametrize("group", [None, 128])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_norm_fp8(dim, group, dtype):
    from gbxcule_amd.rl import rms_norm, rms_norm_fp8

    gen = _gen(dim + 1)
    rows = 9
    x, w, r = _randn(gen, rows, dim, dtype=dtype), 1.0 + _randn(gen, dim, scale=0.2), _randn(gen, rows, dim, dtype=dtype)
    x[3] = 0
    r[3] = 0  # a row of zeros
    q, scale, s = rms_norm_fp8(x, w, r, group=group)
    y, s2 = rms_norm(x.float(), w, None if r is None else (x + r).float() - x.float())
    assert q.dtype is torch.float8_e4m3fn and torch.equal(s, x + r)
    y, _ = ref.rms_norm(ref.f64(x), ref.f64(w), ref.f64(r), 1e-6, dtype)
    size = group or dim
    tops = torch.stack([b.abs().amax(-1) for b in y.split(size, -1)], -1).clamp_min(1e-30)
    ref.check(scale if group else scale.unsqueeze(-1), tops / 448, 16 + 3 * dim.bit_length() + dim // 256, "scale")
    wide = (tops / 448).repeat_interleave(size, dim=-1)[:, :dim]
    back = q.float().cpu().double() * wide
    # e4m3: half a step is 2^-4 of the value, or 2^-10 of the scale below its normal range; one
    # step more next to a boundary
    assert bool(((back - y).abs() <= y.abs() * 2.0**-4 * 1.01 + wide * 2.0**-10 * 1.01 + 1e-12).all())
    assert not q[3].float().any()


def test_norm_special_rows_and_strides():
    from gbxcule_amd.rl import rms_norm, rms_norm_fp8

    gen = _gen(3)
    base = _randn(gen, 6, 5, 300, dtype=BF16)
    w = 1.0 + _randn(gen, 100, scale=0.1)
    for x in (base[..., 100:200], base[..., 1:101], base[::2, 1:4, 7:107], base[..., ::3], base[:, :1, :100].expand(6, 5, 100)):
        y, _ = ref.rms_norm(ref.f64(x), ref.f64(w), None, 1e-6, BF16)
        ref.check(rms_norm(x, w), y, 64, str(x.stride()))
    x = _randn(gen, 4, 512)
    x[1, 7], x[2, 9] = float("nan"), float("inf")
    y = rms_norm(x, torch.ones(512, device="cuda"))
    assert torch.isnan(y[1]).all() and torch.isnan(y[2, 9]) and not y[2, :9].any() and torch.isfinite(y[[0, 3]]).all()
    q, scale = rms_norm_fp8(x, torch.ones(512, device="cuda"), group=128)
    assert torch.isnan(scale[1]).all() and torch.isnan(q[1].float()).all() and torch.isfinite(scale[[0, 3]]).all()
    assert rms_norm(x[:0], torch.ones(512, device="cuda")).shape == (0, 512)
    # a weight in the stream's type gets its gradient in that type
    wb = w.to(BF16).requires_grad_()
    (g,) = torch.autograd.grad(rms_norm(base[0, :, :100], wb).float().sum(), wb)
    assert g.dtype is BF16 and g.shape == (100,)
    # only the sum is used: its gradient goes through
    xs = base[0, :, :100].detach().requires_grad_()
    _, s = rms_norm(xs, w, base[1, :, :100])
    (g,) = torch.autograd.grad(s.float().sum(), xs)
    assert torch.equal(g, torch.ones_like(g))


# ------------------------------------------------------- the causal convolution

CONVS = [
    # steps, envs, dim, width, dtype, resets, bias, silu, state
    (1, 1, 1, 2, F32, 0.0, True, True, True),
    (1, 3, 8, 4, BF16, 1.0, True, True, True),
    (2, 3, 9, 4, F32, 0.5, True, True, True),
    (3, 2, 7, 4, F16, 0.0, False, False, True),
    (15, 4, 16, 3, BF16, 0.2, True, True, False),
    (16, 1, 264, 4, F32, 0.1, True, True, True),
    (17, 5, 33, 4, F32, 0.3, True, False, True),
    (33, 2, 100, 2, BF16, 1.0, False, True, True),
    (50, 3, 65, 4, F32, 0.1, True, True, True),
    (130, 1, 40, 3, F16, 0.02, True, True, True),
    (257, 7, 24, 4, F32, 0.05, True, True, False),
]


@pytest.mark.parametrize("case", CONVS, ids=str)
def test_conv(case):
    from gbxcule_amd.rl import causal_conv, causal_conv_step

    steps, envs, dim, width, dtype, prob, has_bias, silu, has_state = case
    gen = _gen(steps * 31 + dim)
    wide_x = _randn(gen, steps, envs, 2 * dim + 1, dtype=dtype)
    x, w, b = _leaf(wide_x[..., 1 : dim + 1], _randn(gen, dim, width, scale=0.5), _randn(gen, dim) if has_bias else None)
    state = _randn(gen, envs, width - 1, dim, dtype=dtype) if has_state else None
    resets = torch.rand((steps, envs), device="cuda", generator=gen) < prob if prob else None
    act = "silu" if silu else None
    y, last = causal_conv(x, w, b, state=state, resets=resets, activation=act)
    wide = [ref.f64(t) for t in (x, w, b)]
    cpu_resets = None if resets is None else resets.cpu()
    want, want_last = ref.causal_conv(*wide, ref.f64(state), cpu_resets, silu)
    ref.check(y, want, 16, "y")
    assert torch.equal(last.cpu().double(), want_last.detach())
    dy = _randn(gen, envs, steps, dim, dtype=dtype).transpose(0, 1)
    leaves = [t for t in (x, w, b) if t is not None]
    got = torch.autograd.grad(y, leaves, dy)
    exact = torch.autograd.grad(want, [t for t in wide if t is not None], ref.f64(dy))
    ref.check(got[0], exact[0], 32, "gradient of x")
    for g, v, name in zip(got[1:], exact[1:], ("weight", "bias")):
        ref.check(g, v, 32 + steps * envs, f"gradient of {name}")
    # the same rollout one step at a time
    state = torch.zeros(envs, width - 1, dim, dtype=dtype, device="cuda") if state is None else state.clone()
    with torch.no_grad():
        for t in range(steps):
            one = causal_conv_step(x[t], w, b, state, resets=None if resets is None else resets[t], activation=act)
            ref.check(one, want[t], 16, f"step {t}")
    assert torch.equal(state, last)


def test_conv_ignores_what_lies_before_an_episode():
    from gbxcule_amd.rl import causal_conv, causal_conv_step

    gen = _gen(5)
    x, w = _randn(gen, 40, 3, 24), _randn(gen, 24, 4)
    clean = x.clone()
    x[17, 1], x[36, 2] = float("nan"), float("inf")
    resets = torch.zeros(40, 3, dtype=torch.uint8, device="cuda")
    resets[0], resets[18, 1], resets[37, 2] = 1, 255, 2
    state = torch.full((3, 3, 24), float("nan"), device="cuda")
    y, last = causal_conv(x, w, state=state, resets=resets)
    want, want_last = causal_conv(clean, w, resets=resets)
    hit = torch.zeros(40, 3, dtype=torch.bool, device="cuda")
    hit[17, 1] = hit[36, 2] = True
    assert torch.equal(y[~hit], want[~hit]) and not torch.isfinite(y[hit]).any()
    assert torch.equal(last, want_last)
    xs = x.clone().requires_grad_()
    y, _ = causal_conv(xs, w, state=state, resets=resets)
    dy = _randn(gen, 40, 3, 24)
    (g,) = torch.autograd.grad(y, xs, dy)
    cs = clean.clone().requires_grad_()
    (v,) = torch.autograd.grad(causal_conv(cs, w, resets=resets)[0], cs, dy)
    near = hit.clone()  # steps whose own output, or one that they reach, is not finite
    for t, n in ((17, 1), (36, 2)):
        near[t - 3 : t + 1, n] = True
    assert torch.equal(g[~near], v[~near])
    causal_conv_step(x[0], w, None, state, resets=resets[0])
    assert torch.isfinite(state).all() and torch.equal(state[:, 2], x[0]) and not state[:, :2].any()


# ---------------------------------------------------------- the selective scan

SCANS = [
    # steps, envs, dim, states, groups, dtype, resets, gate, skip, bias, softplus, state
    (1, 1, 1, 1, 1, F32, 0.0, True, True, True, True, True),
    (1, 3, 8, 16, 1, BF16, 1.0, True, True, True, True, True),
    (2, 2, 5, 3, 1, F32, 0.5, False, True, False, True, True),
    (15, 2, 63, 8, 1, F32, 0.1, True, True, True, True, True),
    (16, 3, 64, 16, 1, F32, 0.1, True, True, True, True, False),
    (17, 1, 65, 16, 1, F32, 0.1, True, False, True, True, True),
    (33, 2, 130, 16, 1, BF16, 0.1, True, True, True, True, True),
    (48, 3, 40, 32, 1, F32, 0.05, True, True, True, True, True),
    (50, 2, 36, 4, 2, F16, 0.05, True, True, False, False, True),
    (40, 2, 96, 12, 4, F32, 0.0, False, False, False, False, True),
    (70, 1, 100, 24, 2, BF16, 0.02, True, True, True, True, True),
    (100, 5, 34, 5, 2, F32, 1.0, True, True, True, True, True),
    (200, 1, 72, 8, 1, BF16, 0.01, True, True, True, True, True),
    (513, 1, 33, 16, 1, F32, 0.01, True, True, True, True, True),
]
NAMES = ("x", "dt", "A", "B", "C", "D", "z", "dt_bias")


def _scan_inputs(case):
    steps, envs, dim, states, groups, dtype, prob, gate, skip, bias, softplus, has_state = case
    gen = _gen(steps * 17 + dim + states)
    row = _randn(gen, steps, envs, 3 + 2 * groups * states, dtype=dtype)
    cut = lambda at: row[..., at : at + groups * states].unflatten(-1, (groups, states))  # noqa: E731
    raw = _randn(gen, steps, envs, dim, scale=0.7) - 2.0
    t = {
        "x": _randn(gen, steps, envs, dim, dtype=dtype),
        "dt": (raw if softplus else raw.exp()).to(dtype),
        "A": -torch.exp(_randn(gen, dim, states, scale=0.5)),
        "B": cut(3), "C": cut(3 + groups * states),
        "D": _randn(gen, dim) if skip else None,
        "z": _randn(gen, steps, envs, 2 * dim, dtype=dtype)[..., dim:] if gate else None,
        "dt_bias": _randn(gen, dim, scale=0.3).abs() if bias else None,
    }  # fmt: skip
    state = _randn(gen, envs, dim, states) if has_state else None
    resets = torch.rand((steps, envs), device="cuda", generator=gen) < prob if prob else None
    return gen, t, state, resets


@pytest.mark.parametrize("case", SCANS, ids=str)
def test_scan(case):
    from gbxcule_amd.rl import selective_scan, selective_scan_step

    steps, envs, dim, states, groups, dtype, softplus = *case[:6], case[10]
    gen, t, state, resets = _scan_inputs(case)
    leaf = dict(zip(NAMES, _leaf(*(t[k] for k in NAMES))))
    dt_bias = leaf["dt_bias"]
    args = [leaf[k] for k in NAMES[:7]]
    y, last = selective_scan(*args, dt_bias=dt_bias, softplus=softplus, state=state, resets=resets)
    wide = {k: ref.f64(leaf[k]) for k in NAMES}
    want, want_last = ref.selective_scan(*(wide[k] for k in NAMES), softplus, ref.f64(state), None if resets is None else resets.cpu())
    # a state sums the steps that its decay (a few dozen steps at the sizes here) reaches
    n = 128 + steps
    ref.check(y, want, n, "y")
    ref.check(last, want_last, n, "state")
    with torch.no_grad():  # the form without a gradient gives the same
        y2, last2 = selective_scan(*args, dt_bias=dt_bias, softplus=softplus, state=state, resets=resets)
    assert torch.equal(y, y2) and torch.equal(last, last2)
    dy = _randn(gen, envs, steps, dim, dtype=dtype).transpose(0, 1)
    names = [k for k in NAMES if leaf[k] is not None]
    got = torch.autograd.grad(y, [leaf[k] for k in names], dy)
    exact = torch.autograd.grad(want, [wide[k] for k in names], ref.f64(dy))
    for g, v, name in zip(got, exact, names):
        ref.check(g, v, 2 * n + (steps * envs if name in ("A", "D", "dt_bias") else dim), f"gradient of {name}")
    # the same rollout one step at a time
    state = torch.zeros(envs, dim, states, device="cuda") if state is None else state.clone()
    with torch.no_grad():
        for i in range(steps):
            row = [leaf[k][i] if k in ("x", "dt", "B", "C") or (k == "z" and leaf[k] is not None) else leaf[k] for k in NAMES[:7]]
            one = selective_scan_step(*row, state=state, dt_bias=dt_bias, softplus=softplus, resets=None if resets is None else resets[i])
            ref.check(one, want[i], n, f"step {i}")
    ref.check(state, want_last, n, "state after the steps")


def test_scan_pieces_join_as_one():
    """A row cut along the steps gives what it gives in two calls."""
    from gbxcule_amd.rl import selective_scan

    case = (1000, 1, 96, 16, 1, F32, 0.003, True, True, True, True, True)
    _, t, state, resets = _scan_inputs(case)
    args = [t[k] for k in NAMES[:7]]
    y, last = selective_scan(*args, dt_bias=t["dt_bias"], state=state, resets=resets)
    part = lambda a, b: [v[a:b] if k in ("x", "dt", "B", "C", "z") else v for k, v in zip(NAMES, args)]  # noqa: E731
    y1, mid = selective_scan(*part(0, 333), dt_bias=t["dt_bias"], state=state, resets=resets[:333])
    y2, end = selective_scan(*part(333, 1000), dt_bias=t["dt_bias"], state=mid, resets=resets[333:])
    ref.check(torch.cat([y1, y2]), y, 256, "y")
    ref.check(end, last, 256, "state")


@pytest.mark.parametrize("case", [
    (1100, 1, 70, 16, 1, F32, 0.004, True, True, True, True, True),
    (1537, 2, 65, 8, 1, BF16, 0.01, True, True, True, True, True),
    (4801, 1, 33, 4, 1, F32, 0.0, False, True, True, True, True),
], ids=str)  # fmt: skip
def test_scan_of_many_pieces(case):
    """One long row: 64 pieces and more than 256, which are joined by runs."""
    from gbxcule_amd.rl import selective_scan

    steps, envs, dim, states, groups, dtype = case[:6]
    gen, t, state, resets = _scan_inputs(case)
    leaf = dict(zip(NAMES, _leaf(*(t[k] for k in NAMES))))
    y, last = selective_scan(*(leaf[k] for k in NAMES[:7]), dt_bias=leaf["dt_bias"], state=state, resets=resets)
    wide = {k: ref.f64(leaf[k]) for k in NAMES}
    want, want_last = ref.selective_scan(*(wide[k] for k in NAMES), True, ref.f64(state), None if resets is None else resets.cpu())
    # the roundings that a state carries are those of the steps that its decay reaches, joins of pieces among them
    n = 512
    ref.check(y, want, n, "y")
    ref.check(last, want_last, n, "state")
    dy = _randn(gen, steps, envs, dim, dtype=dtype)
    names = [k for k in NAMES if leaf[k] is not None]
    got = torch.autograd.grad(y, [leaf[k] for k in names], dy)
    exact = torch.autograd.grad(want, [wide[k] for k in names], ref.f64(dy))
    for g, v, name in zip(got, exact, names):
        ref.check(g, v, 2 * n + (steps * envs if name in ("A", "D", "dt_bias") else dim), f"gradient of {name}")


@pytest.mark.parametrize("steps", [40, 400])
def test_scan_ignores_what_lies_before_an_episode(steps):
    from gbxcule_amd.rl import selective_scan, selective_scan_step

    case = (steps, 2, 70, 16, 1, F32, 0.0, True, True, True, True, False)
    gen, t, _, _ = _scan_inputs(case)
    resets = torch.zeros(steps, 2, dtype=torch.bool, device="cuda")
    resets[0] = resets[19, 1] = True
    state = torch.full((2, 70, 16), float("nan"), device="cuda")
    dy = _randn(gen, steps, 2, 70)

    def both(x, state):
        leaf = _leaf(x, t["dt"], t["B"], t["C"], t["z"])
        y, last = selective_scan(leaf[0], leaf[1], t["A"], leaf[2], leaf[3], t["D"], leaf[4], dt_bias=t["dt_bias"],
                                 state=state, resets=resets)  # fmt: skip
        return [y.detach(), *torch.autograd.grad(y, leaf, dy)], last

    want, want_last = both(t["x"], None)
    x = t["x"].clone()
    x[18, 1] = float("nan")
    got, last = both(x, state)
    assert torch.equal(last, want_last)
    fine = torch.ones(steps, 2, dtype=torch.bool, device="cuda")
    fine[18, 1] = False
    assert torch.isnan(got[0][18, 1]).all()
    fine_before = fine.clone()
    for g, w in zip(got, want):
        assert torch.equal(g[fine_before], w[fine_before])
    row = [v[0] for v in (x, t["dt"], t["B"], t["C"], t["z"])]
    with torch.no_grad():
        y = selective_scan_step(row[0], row[1], t["A"], row[2], row[3], t["D"], row[4], state=state, dt_bias=t["dt_bias"], resets=resets[0])
    assert torch.isfinite(state).all() and torch.isfinite(y).all()


@pytest.mark.parametrize("op", ["norm", "conv", "scan"])
def test_gradients_against_differences(op):
    """Central differences of the kernels' own outputs along one direction per
    input.  The sum of y * dy over about 2,000 outputs of size 1 is right to
    2^-23 * sqrt(2000) * 4, divided by 2 eps = 0.02: 1e-3; the third derivative
    adds eps^2 = 1e-4 of a gradient of size 50."""
    from gbxcule_amd.rl import causal_conv, rms_norm, selective_scan

    gen = _gen(11)
    resets = torch.rand((20, 3), device="cuda", generator=gen) < 0.1
    if op == "norm":
        tensors = [_randn(gen, 60, 33), 1 + _randn(gen, 33, scale=0.1), _randn(gen, 60, 33)]
        f = lambda x, w, r: rms_norm(x, w, r)[0]  # noqa: E731
    elif op == "conv":
        tensors = [_randn(gen, 20, 3, 33), _randn(gen, 33, 4), _randn(gen, 33)]
        f = lambda x, w, b: causal_conv(x, w, b, resets=resets)[0]  # noqa: E731
    else:
        _, t, _, _ = _scan_inputs((20, 3, 33, 16, 1, F32, 0.0, True, True, True, True, False))
        tensors = [t[k] for k in NAMES]
        f = lambda *a: selective_scan(*a[:7], dt_bias=a[7], resets=resets)[0]  # noqa: E731
    dy = None
    for i in range(len(tensors)):
        leaves = _leaf(*tensors)
        y = f(*leaves)
        dy = _randn(gen, *y.shape) if dy is None else dy
        (g,) = torch.autograd.grad(y, leaves[i], dy)
        v = _randn(gen, *tensors[i].shape)
        v /= v.norm()
        eps = 0.01
        moved = [[t + s * eps * v if k == i else t for k, t in enumerate(tensors)] for s in (1, -1)]
        with torch.no_grad():
            slope = ((f(*moved[0]).double() - f(*moved[1]).double()) * dy.double()).sum() / (2 * eps)
        want = (g.double() * v.double()).sum()
        assert abs(float(slope - want)) <= 1e-3 + 1e-4 * 50 + 1e-3 * abs(float(want)), (op, i, float(slope), float(want))


# ------------------------------------------------- offsets, streams, refusals


def test_offsets_beyond_32_bits():
    """Rollouts and states of more than 2^31 elements: the last envs give what
    they give alone."""
    from gbxcule_amd.rl import causal_conv, rms_norm, selective_scan, selective_scan_step

    gen = _gen(2)
    steps, envs, dim = 17, 131_072, 1024
    x = torch.empty(steps, envs, dim, dtype=BF16, device="cuda").normal_(generator=gen)
    w = _randn(gen, dim, 4)
    tail = slice(envs - 2, envs)
    with torch.no_grad():
        y, last = causal_conv(x, w)
        y1, last1 = causal_conv(x[:, tail], w)
        assert torch.equal(y[:, tail], y1) and torch.equal(last[tail], last1)
        y = rms_norm(x, w[:, 0].contiguous())
        assert torch.equal(y[:, tail], rms_norm(x[:, tail], w[:, 0].contiguous()))
        del y, y1
    A = -torch.exp(_randn(gen, dim, 16))
    bc = _randn(gen, steps, envs, 32, dtype=BF16)
    dt = x  # any step sizes do

    def scan(part):
        xs, dts = _leaf(x[:, part], dt[:, part])
        y, last = selective_scan(xs, dts, A, bc[:, part, :16], bc[:, part, 16:])
        (g,) = torch.autograd.grad(y, xs, xs.detach())
        return y[:, -2:].detach().clone(), last[-2:].clone(), g[:, -2:].clone()

    for big, small in zip(scan(slice(0, envs)), scan(tail)):
        ref.check(big, small, 256)
    del x, dt
    torch.cuda.empty_cache()
    state = torch.empty(envs, dim, 32, device="cuda").normal_(generator=gen)
    kept = state[tail].clone()
    A = -torch.exp(_randn(gen, dim, 32))
    one, bc = _randn(gen, envs, dim, dtype=BF16), _randn(gen, envs, 64, dtype=BF16)
    with torch.no_grad():
        y = selective_scan_step(one, one, A, bc[:, :32], bc[:, 32:], state=state)
        y1 = selective_scan_step(one[tail], one[tail], A, bc[tail, :32], bc[tail, 32:], state=kept)
    assert torch.equal(y[tail], y1) and torch.equal(state[tail], kept)


def test_empty_rollouts():
    from gbxcule_amd.rl import causal_conv, causal_conv_step, rms_norm_fp8, selective_scan, selective_scan_step

    z = lambda *s: torch.zeros(s, device="cuda")  # noqa: E731
    state = torch.rand(3, 8, 16, device="cuda")
    y, last = selective_scan(z(0, 3, 8), z(0, 3, 8), z(8, 16), z(0, 3, 16), z(0, 3, 16), state=state)
    assert y.shape == (0, 3, 8) and torch.equal(last, state) and last.data_ptr() != state.data_ptr()
    y, last = selective_scan(z(4, 0, 8), z(4, 0, 8), z(8, 16), z(4, 0, 16), z(4, 0, 16))
    assert y.shape == (4, 0, 8) and last.shape == (0, 8, 16)
    assert selective_scan_step(z(0, 8), z(0, 8), z(8, 16), z(0, 16), z(0, 16), state=z(0, 8, 16)).shape == (0, 8)
    window = torch.rand(3, 3, 8, device="cuda")
    y, last = causal_conv(z(0, 3, 8), z(8, 4), state=window)
    assert y.shape == (0, 3, 8) and torch.equal(last, window)
    assert causal_conv_step(z(0, 8), z(8, 4), None, z(0, 3, 8)).shape == (0, 8)
    q, scale = rms_norm_fp8(z(0, 300), torch.ones(300, device="cuda"), group=128)
    assert q.shape == (0, 300) and scale.shape == (0, 3)


def test_other_streams_and_capture():
    from gbxcule_amd.rl import causal_conv_step, rms_norm_fp8, selective_scan, selective_scan_step

    case = (60, 2, 64, 16, 1, BF16, 0.1, True, True, True, True, True)
    gen, t, state, resets = _scan_inputs(case)
    args = [t[k] for k in NAMES[:7]]
    want = selective_scan(*args, dt_bias=t["dt_bias"], state=state, resets=resets)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = selective_scan(*args, dt_bias=t["dt_bias"], state=state, resets=resets)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])

    # the actor's step as a graph: every replay moves the states on as eager calls do
    row = [v[0].contiguous() if k in ("x", "dt", "B", "C", "z") else v for k, v in zip(NAMES, args)]
    w, nw = _randn(gen, 64, 4), 1 + _randn(gen, 64, scale=0.1)
    window, h = _randn(gen, 2, 3, 64, dtype=BF16), state.clone()
    window2, h2 = window.clone(), h.clone()

    def step(window, h):
        u = causal_conv_step(row[0], w, None, window)
        y = selective_scan_step(u, *row[1:], state=h, dt_bias=t["dt_bias"])
        return rms_norm_fp8(y, nw)

    with torch.no_grad():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            q, scale = step(window, h)
        for k in range(4):
            row[0].copy_(_randn(gen, 2, 64, dtype=BF16))
            graph.replay()
            torch.cuda.synchronize()
            q2, scale2 = step(window2, h2)
            assert torch.equal(h, h2) and torch.equal(window, window2), k
            assert torch.equal(q.float(), q2.float()) and torch.equal(scale, scale2), k


def test_refusals():
    from gbxcule_amd.rl import causal_conv, causal_conv_step, rms_norm, rms_norm_fp8, selective_scan, selective_scan_step

    z = lambda *s, **k: torch.zeros(s, device="cuda", **k)  # noqa: E731
    x, w = z(4, 3, 8), z(8)

    def refused(f, *a, error=ValueError, **k):
        with pytest.raises(error):
            f(*a, **k)

    refused(rms_norm, x.cpu(), w)
    refused(rms_norm, x.double(), w)
    refused(rms_norm, [1.0], w, error=TypeError)
    refused(rms_norm, x, z(9))
    refused(rms_norm, x, w.cpu())
    refused(rms_norm, x, w, z(4, 3, 7))
    refused(rms_norm, x, w, x.half())
    refused(rms_norm_fp8, x, w, group=64)
    refused(rms_norm_fp8, x.clone().requires_grad_(), w, error=RuntimeError)
    refused(causal_conv, x[0], z(8, 4))
    refused(causal_conv, x, z(8, 5))
    refused(causal_conv, x, z(8, 1))
    refused(causal_conv, x, z(7, 4))
    refused(causal_conv, x, z(8, 4), z(7))
    refused(causal_conv, x, z(8, 4), state=z(3, 2, 8))
    refused(causal_conv, x, z(8, 4), state=z(3, 3, 8, dtype=BF16))
    refused(causal_conv, x, z(8, 4), state=z(3, 3, 8).requires_grad_())
    refused(causal_conv, x, z(8, 4), resets=z(3, 4, dtype=torch.bool))
    refused(causal_conv, x, z(8, 4), resets=z(4, 3))
    refused(causal_conv, x, z(8, 4), activation="relu")
    refused(causal_conv_step, x[0], z(8, 4), None, z(3, 8, 3).transpose(1, 2))
    refused(causal_conv_step, x[0].clone().requires_grad_(), z(8, 4), None, z(3, 3, 8), error=RuntimeError)
    ok = dict(dt=x, A=z(8, 16), B=z(4, 3, 16), C=z(4, 3, 16))
    selective_scan(x, **ok)
    for bad in (dict(dt=x[:2]), dict(dt=x.half()), dict(A=z(8, 33), B=z(4, 3, 33), C=z(4, 3, 33)), dict(A=z(7, 16)),
                dict(B=z(4, 3, 15)), dict(C=z(4, 2, 16)), dict(B=z(4, 3, 3, 16), C=z(4, 3, 3, 16)),
                dict(C=z(4, 3, 2, 16)), dict(D=z(7)), dict(z=x[:1]), dict(dt_bias=z(7)), dict(state=z(3, 8, 15)),
                dict(state=z(3, 8, 16, dtype=BF16)), dict(state=z(3, 8, 16).requires_grad_()),
                dict(resets=z(4, 2, dtype=torch.bool)), dict(A=z(8, 0), B=z(4, 3, 0), C=z(4, 3, 0))):  # fmt: skip
        refused(selective_scan, x, **{**ok, **bad})
    row = dict(dt=x[0], A=z(8, 16), B=z(3, 16), C=z(3, 16))
    refused(selective_scan_step, x[0], **row, state=z(3, 16, 8).transpose(1, 2))
    refused(selective_scan_step, x[0], **row, state=z(2, 8, 16))
    refused(selective_scan_step, x[0].clone().requires_grad_(), **row, state=z(3, 8, 16), error=RuntimeError)
