"""The gated delta rule against its plain 64-bit form, step by step: sizes around
every tile and chunk, types, shared heads, strides, episode starts and closed
gates, values behind them that must not be seen, keys that repeat, gradients
against autograd and against differences, single steps against whole rollouts,
streams, graphs, and refusals."""

from __future__ import annotations

import math

import pytest
import torch

from . import _policy_ref as ref
from .conftest import require_gpu

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
NAMES = ("q", "k", "v", "g", "beta")


@pytest.fixture(autouse=True)
def _gpu():
    require_gpu()


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape, dtype=F32, scale=1.0):
    return (torch.randn(shape, device="cuda", generator=gen) * scale).to(dtype)


def _rand(gen, *shape):
    return torch.rand(shape, device="cuda", generator=gen)


def _inputs(seed, steps, envs, heads, keys, values, share=1, dtype=F32, resets=0.0, normalize=True, state=True):
    gen = _gen(seed)
    s = {"q": _randn(gen, steps, envs, heads // share, keys, dtype=dtype), "k": _randn(gen, steps, envs, heads // share, keys, dtype=dtype)}
    if not normalize:
        s["q"], s["k"] = s["q"] * keys**-0.5, s["k"] * (0.8 * keys**-0.5)
    s["v"] = _randn(gen, steps, envs, heads, values, dtype=dtype)
    s["g"] = -0.02 - 0.4 * _rand(gen, steps, envs, heads)
    s["beta"] = torch.sigmoid(_randn(gen, steps, envs, heads))
    s["state"] = _randn(gen, envs, heads, keys, values, scale=0.5) if state else None
    s["resets"] = _rand(gen, steps, envs) < resets if resets else None
    s["dy"] = _randn(gen, steps, envs, heads, values, dtype=dtype)
    return s


def _plain(q, k, v, g, beta, state, resets, normalize=True, scale=None):
    """64 bits, one step after the other."""
    steps, envs, heads, values = v.shape
    share, keys = heads // q.shape[2], q.shape[3]
    if normalize:
        q, k = (t / torch.sqrt((t * t).sum(-1, keepdim=True) + 1e-6) for t in (q, k))
    q, k = (t.repeat_interleave(share, dim=2) for t in (q, k))
    scale = keys**-0.5 if scale is None else scale
    S = torch.zeros(envs, heads, keys, values, dtype=torch.float64) if state is None else state
    out = []
    for t in range(steps):
        cut = g[t] < -104.0
        if resets is not None:
            cut = cut | (resets[t, :, None] != 0)
        S = torch.where(cut[..., None, None], 0.0, torch.exp(g[t])[..., None, None] * S)
        e = beta[t][..., None] * (v[t] - (S * k[t][..., None]).sum(-2))
        S = S + k[t][..., None] * e[..., None, :]
        out.append(scale * (S * q[t][..., None]).sum(-2))
    return torch.stack(out) if out else v.new_zeros(v.shape), S


def _roundings(steps, keys):
    """Each step's products sum over the keys, four lanes' parts and four
    places each, and over the 16 steps of a chunk; the state carries what is
    off through all steps, since what it forgets makes errors smaller too."""
    return 32 + keys // 2 + 2 * steps


def _leaves(s):
    return [s[k].detach().requires_grad_() for k in NAMES]


def _terms(wide, s, scale):
    """The size of what the gradient of a row's length subtracts: (d - u (u . d)) / length, with d that of the row u of
    unit length, is as small as the row is long along d, and with one channel next to nothing; its roundings are of d / length."""
    units, sizes = [], []
    for t in wide[:2]:
        size = torch.sqrt((t.detach() ** 2).sum(-1, keepdim=True) + 1e-6)
        units.append((t.detach() / size).requires_grad_())
        sizes.append(size)
    y, _ = _plain(*units, *(t.detach() for t in wide[2:]), ref.f64(s["state"]), None if s["resets"] is None else s["resets"].cpu(), False, scale)
    found = torch.autograd.grad(y, units, ref.f64(s["dy"]))
    return {name: float((d / size).abs().max()) for name, d, size in zip("qk", found, sizes)}


def _check_terms(got, want, roundings, terms, what):
    """``ref.check`` with roundings of the size of the largest term, where that is more than the largest value."""
    want, got = want.detach().cpu().double(), got.detach().cpu()
    big = max(float(want.abs().max()), terms)
    atol = roundings * 2.0**-23 * big + ref.FLOOR[got.dtype] + 1e-30
    torch.testing.assert_close(got.double(), want, rtol=ref.UNIT[got.dtype], atol=atol, msg=lambda m: f"{what}: {m}")


def _compare(s, normalize=True, scale=None):
    from gbxcule_amd.rl import delta_rule

    leaves = _leaves(s)
    wide = [ref.f64(t) for t in leaves]
    y, last = delta_rule(*leaves, state=s["state"], resets=s["resets"], normalize=normalize, scale=scale)
    want, want_last = _plain(*wide, ref.f64(s["state"]), None if s["resets"] is None else s["resets"].cpu(), normalize, scale)
    steps, keys = s["q"].shape[0], s["q"].shape[3]
    n = _roundings(steps, keys)
    ref.check(y, want, n, "y")
    ref.check(last, want_last, n, "state")
    assert not last.requires_grad
    got = torch.autograd.grad(y, leaves, s["dy"])
    exact = torch.autograd.grad(want, wide, ref.f64(s["dy"]))
    for a, b, name in zip(got, exact, NAMES):
        # a gradient goes through the forward's roundings, its own way back, and sums over the channels
        _check_terms(a, b, 4 * n + s["v"].shape[3], _terms(wide, s, scale)[name] if normalize and name in "qk" else 0.0, f"gradient of {name}")
    with torch.no_grad():
        again = delta_rule(*leaves, state=s["state"], resets=s["resets"], normalize=normalize, scale=scale)
    assert torch.equal(again[0], y) and torch.equal(again[1], last)
    return y, last, got


CASES = [
    # steps, envs, heads, keys, values, share, dtype, resets, normalize, state
    (1, 1, 1, 1, 1, 1, F32, 0.0, True, True),
    (1, 3, 2, 64, 64, 1, BF16, 1.0, True, True),
    (2, 2, 2, 8, 5, 2, F32, 0.5, True, True),
    (15, 2, 1, 16, 16, 1, F32, 0.0, True, False),
    (16, 2, 3, 32, 32, 1, BF16, 0.0, True, True),
    (17, 1, 2, 33, 31, 1, F32, 0.2, True, True),
    (16, 3, 1, 64, 64, 1, F32, 0.0, False, True),
    (31, 2, 2, 64, 65, 2, F16, 0.1, True, True),
    (33, 2, 4, 40, 56, 4, F32, 0.05, True, True),
    (48, 1, 1, 63, 17, 1, BF16, 0.1, False, False),
    (50, 2, 2, 128, 128, 1, BF16, 0.02, True, True),
    (20, 1, 2, 127, 100, 2, F32, 0.1, True, True),
    (40, 1, 1, 65, 128, 1, F16, 0.0, True, True),
    (19, 2, 1, 3, 128, 1, F32, 1.0, True, True),
    (21, 2, 2, 128, 2, 1, F32, 0.3, False, True),
    (100, 3, 2, 24, 48, 1, BF16, 0.05, True, True),
    (200, 2, 1, 64, 64, 1, F32, 0.01, True, True),
    # few heads and many steps, which are cut into pieces
    (256, 1, 1, 64, 64, 1, F32, 0.0, True, True),
    (700, 1, 2, 40, 24, 2, F32, 0.005, True, True),
    (555, 2, 1, 128, 100, 1, BF16, 0.01, True, False),
    (430, 1, 3, 32, 48, 1, F16, 0.0, True, True),
    (321, 1, 1, 100, 128, 1, F32, 0.02, False, True),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_against_steps(case):
    steps, envs, heads, keys, values, share, dtype, resets, normalize, state = case
    _compare(_inputs(steps * 7 + keys, steps, envs, heads, keys, values, share, dtype, resets, normalize, state), normalize)


def test_scale():
    _compare(_inputs(5, 20, 2, 2, 24, 24), scale=0.7)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_the_same_key_at_every_step(dtype):
    """A screen that stands still: the system's rows are all alike, and every correction undoes most of the one before."""
    s = _inputs(6, 70, 2, 2, 64, 64, dtype=dtype)
    s["k"] = s["k"][:1].expand_as(s["k"]).contiguous()
    s["q"] = s["q"][:1].expand_as(s["q"]).contiguous()
    s["beta"] = torch.full_like(s["beta"], 0.97)
    _compare(s)


def test_closed_and_open_gates():
    """Gates from 0 to -infinity; those below -104 clear the state, and what they say of its gradient is nothing."""
    s = _inputs(7, 40, 2, 2, 16, 24)
    s["g"][5], s["g"][6], s["g"][17, 0], s["g"][30] = -104.5, -math.inf, -1e30, -100.0
    s["g"][8:12] = 0.0
    s["g"][20:23] = -60.0
    wide_g = s["g"].clone()
    *_, got = _compare({**s, "g": wide_g.clamp_min(-1e30)})
    assert not got[3][5].any() and not got[3][6].any() and not got[3][17, 0].any() and torch.isfinite(got[3]).all()
    from gbxcule_amd.rl import delta_rule

    rows = [s[k] for k in NAMES]
    y, last = delta_rule(*rows, state=s["state"])
    rows[3] = wide_g.clamp_min(-1e30)
    y2, last2 = delta_rule(*rows, state=s["state"])
    assert torch.equal(y, y2) and torch.equal(last, last2) and torch.isfinite(y).all()


def test_strides_and_gate_types():
    """q, k and v as parts of one projection's output, in another order of
    dimensions, shared by all envs; gates in 16 bits; a gradient that is one
    number for all."""
    from gbxcule_amd.rl import delta_rule

    gen = _gen(8)
    steps, envs, heads, d = 23, 3, 2, 40
    wide = _randn(gen, steps, envs, heads * 3 * d + 5, dtype=BF16)
    q, k, v = (t.unflatten(-1, (heads, d)) for t in wide[..., 1 : 1 + heads * 3 * d].split(heads * d, -1))
    g, beta = (-_rand(gen, steps, envs, heads)).to(BF16), _rand(gen, envs, steps, heads).transpose(0, 1)
    turned = _randn(gen, heads, envs, d, steps, dtype=BF16).permute(3, 1, 0, 2)
    for rows in ((q, k, v, g, beta), (turned, k, turned, g, beta), (q[:, :1].expand_as(q), k[:, :, :1].expand_as(k), v, g, beta[:, :, :1].expand_as(beta))):
        leaves = [t.detach().requires_grad_() for t in rows]
        wide_leaves = [ref.f64(t) for t in leaves]
        y, last = delta_rule(*leaves)
        want, want_last = _plain(*wide_leaves, None, None)
        ref.check(y, want, _roundings(steps, d), "y")
        ref.check(last, want_last, _roundings(steps, d), "state")
        got = torch.autograd.grad(y.sum(), leaves)
        exact = torch.autograd.grad(want.sum(), wide_leaves)
        for a, b, leaf, name in zip(got, exact, leaves, NAMES):
            assert a.dtype is leaf.dtype
            ref.check(a, b, 4 * _roundings(steps, d) + d, f"gradient of {name}")


def test_steps_equal_the_rollout():
    from gbxcule_amd.rl import delta_rule, delta_rule_step

    for seed, (envs, heads, keys, values, share, dtype) in enumerate(
        [(5, 4, 64, 64, 2, F32), (3, 1, 33, 47, 1, F32), (2, 2, 128, 100, 1, BF16), (7, 3, 16, 8, 3, F16), (1, 1, 1, 1, 1, F32)]
    ):
        s = _inputs(seed, 18, envs, heads, keys, values, share, dtype, resets=0.2)
        s["g"][4, 0] = -200.0
        rows = [s[k] for k in NAMES]
        y, last = delta_rule(*rows, state=s["state"], resets=s["resets"])
        want, want_last = _plain(*(ref.f64(t) for t in rows), ref.f64(s["state"]), s["resets"].cpu())
        state = s["state"].clone()
        for t in range(18):
            one = delta_rule_step(*(r[t] for r in rows), state=state, resets=s["resets"][t])
            ref.check(one, want[t], _roundings(t + 1, keys), f"step {t}")
        ref.check(state, want_last, _roundings(18, keys), "state")
        ref.check(last, want_last, _roundings(18, keys), "the rollout's state")


def test_nothing_from_before_an_episode():
    """Whatever stands before an episode's start, finite or not, is not in it."""
    from gbxcule_amd.rl import delta_rule, delta_rule_step

    for at in (3, 16, 21):
        s = _inputs(30 + at, 36, 3, 2, 24, 24, share=2)
        s["resets"] = torch.zeros(36, 3, dtype=torch.uint8, device="cuda")
        s["resets"][at] = 1
        rows = [s[k] for k in NAMES]
        dirty = [r.clone() for r in rows]
        for r, bad in zip(dirty, (math.nan, math.inf, -math.inf, math.nan, math.inf)):
            r[:at, 1] = bad
        dirty[3][at, 1] = math.nan  # the gate of the step that begins it, too
        state = s["state"].clone()
        state[1] = math.nan
        y, last = delta_rule(*rows, state=s["state"], resets=s["resets"])
        leaves = [r.requires_grad_() for r in dirty]
        y2, last2 = delta_rule(*leaves, state=state, resets=s["resets"])
        assert torch.equal(y[at:], y2[at:]) and torch.equal(last, last2)
        dy = s["dy"].clone()
        dy[:at] = 0
        got = torch.autograd.grad(y2, leaves, dy)
        clean = [r.detach().requires_grad_() for r in rows]
        want = torch.autograd.grad(delta_rule(*clean, state=s["state"], resets=s["resets"])[0], clean, dy)
        for a, b, name in zip(got, want, NAMES):
            # a rollout with a value that is not finite is walked back span by span, with u computed anew where the
            # other has the forward pass's: two orders of the same sums, each within _roundings of the formulas
            assert float((a[at:] - b[at:]).abs().max()) <= 2 * 4 * _roundings(36, 24) * 2.0**-23 * float(b.abs().max()), name
        one = delta_rule_step(*(r.detach()[at] for r in dirty), state=state, resets=s["resets"][at])
        ref.check(one, ref.f64(y[at]), 64, "step")
        assert torch.isfinite(state).all()


def test_a_value_that_is_not_finite_reaches_later_steps_alone():
    """Before it, outputs and the gradients that the formulas keep from it are what they are without it."""
    from gbxcule_amd.rl import delta_rule

    at = 9
    s = _inputs(40, 30, 2, 2, 24, 40)
    rows = [s[k] for k in NAMES]
    y, last = delta_rule(*rows, state=s["state"])
    for which, bad in ((0, math.nan), (1, math.inf), (2, math.nan), (2, math.inf), (4, math.nan), (3, math.nan)):
        dirty = [r.clone() for r in rows]
        dirty[which][at, 0].view(-1)[1] = bad
        y2, last2 = delta_rule(*dirty, state=s["state"])
        assert torch.equal(y[:, 1], y2[:, 1]) and torch.equal(last[1], last2[1])
        # earlier steps are solved one by one where a later one is not finite: another order of the same sums
        assert float((y2[:at, 0] - y[:at, 0]).abs().max()) <= _roundings(at, 24) * 2.0**-23 * float(y.abs().max())
        if which == 0:  # a query is not remembered
            assert torch.isfinite(y2[at + 1 :]).all() and torch.isfinite(last2).all()
        else:
            assert not torch.isfinite(last2[0]).all()
    # one value of v at the end of a rollout, whose own y the loss leaves out: its column alone goes wrong, and
    # the steps before it have their gradients
    v = s["v"].clone()
    v[at, 0, 1, 5] = math.nan
    dy = s["dy"].clone()
    dy[at:] = 0
    leaves = [t.detach().requires_grad_() for t in (*rows[:2], v, *rows[3:])]
    got = torch.autograd.grad(delta_rule(*leaves, state=s["state"])[0], leaves, dy)
    clean = [t.detach().requires_grad_() for t in rows]
    want = torch.autograd.grad(delta_rule(*clean, state=s["state"])[0], clean, dy)
    for a, b, name in zip(got, want, NAMES):
        assert float((a[:at] - b[:at]).abs().max()) <= 4 * _roundings(30, 24) * 2.0**-23 * float(b.abs().max()), name


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("which", range(5))
def test_a_value_that_is_not_finite_at_any_step_of_a_chunk(which, dtype):
    """The last step of a chunk, whose system does not reach it, as well as the first."""
    from gbxcule_amd.rl import delta_rule

    s = _inputs(41, 19, 1, 2, 24, 40, dtype=dtype)
    rows = [s[k] for k in NAMES]
    clean = [t.detach().requires_grad_() for t in rows]
    y, _ = delta_rule(*clean, state=s["state"])
    near = (_roundings(19, 24) * 2.0**-23 + 2 * ref.UNIT[dtype]) * float(y.detach().abs().max())
    for at in range(19):
        for bad in (math.nan, math.inf):
            dirty = [t.detach().clone() for t in rows]
            dirty[which][at].view(-1)[0] = bad
            leaves = [t.requires_grad_() for t in dirty]
            y2, _ = delta_rule(*leaves, state=s["state"])
            assert not torch.isfinite(y2[at]).all()
            if at:
                assert float((y2[:at] - y[:at]).detach().abs().max()) <= near, (at, bad)
            if which == 0 and at < 18:  # no later step's gradient asks for an earlier query
                assert float((y2[at + 1 :] - y[at + 1 :]).detach().abs().max()) <= near, (at, bad)
                found = torch.autograd.grad(y2, leaves, s["dy"])
                want = torch.autograd.grad(y, clean, s["dy"], retain_graph=True)
                for a, b, name in zip(found, want, NAMES):
                    off = (4 * _roundings(19, 24) * 2.0**-23 + 2 * ref.UNIT[b.dtype]) * float(b.abs().max())
                    assert float((a[at + 1 :] - b[at + 1 :]).abs().max()) <= off, (at, bad, name)


def test_pieces_and_what_is_not_finite():
    """Few heads and many steps: what a value that is not finite reaches, and what an episode's start keeps from it."""
    from gbxcule_amd.rl import delta_rule

    steps, keys = 520, 32
    s = _inputs(60, steps, 2, 1, keys, 24)
    s["resets"] = torch.zeros(steps, 2, dtype=torch.bool, device="cuda")
    s["resets"][300, 1] = True
    rows = [s[k] for k in NAMES]
    y, last = delta_rule(*rows, state=s["state"], resets=s["resets"])
    near = _roundings(steps, keys) * 2.0**-23 * float(y.abs().max())
    for which, at, bad in ((0, 200, math.nan), (1, 7, math.inf), (2, 290, math.nan), (3, 130, math.nan), (4, 299, math.inf), (2, 500, math.inf)):
        dirty = [r.clone() for r in rows]
        dirty[which][at, 1].view(-1)[0] = bad
        y2, last2 = delta_rule(*dirty, state=s["state"], resets=s["resets"])
        assert torch.equal(y2[:, 0], y[:, 0]) and torch.equal(last2[0], last[0])  # the other env
        assert float((y2[:at, 1] - y[:at, 1]).abs().max()) <= near
        assert not torch.isfinite(y2[at : at + 1, 1]).all()
        if at < 300:  # the episode after it
            assert float((y2[300:, 1] - y[300:, 1]).abs().max()) <= near
            assert float((last2[1] - last[1]).abs().max()) <= _roundings(steps, keys) * 2.0**-23 * float(last.abs().max())
    state = s["state"].clone()
    state[1, 0, 3, 5] = math.nan  # one column, until the episode ends
    y2, last2 = delta_rule(*rows, state=state, resets=s["resets"])
    assert torch.isnan(y2[:300, 1, 0, 5]).all() and torch.isfinite(y2[:, 1, 0, 6:]).all() and torch.isfinite(last2).all()
    assert float((y2[300:] - y[300:]).abs().max()) <= near
    # nothing grows from a state of zero, however open the gates: without steps that write there is nothing
    rows[3], rows[4] = torch.full_like(rows[3], 2.0), torch.zeros_like(rows[4])
    y2, last2 = delta_rule(*rows)
    assert not y2.any() and not last2.any()


def test_gradient_against_differences():
    from gbxcule_amd.rl import delta_rule

    s = _inputs(9, 37, 2, 2, 20, 28, share=2, resets=0.05)
    gen = _gen(10)
    rows = [s[k] for k in NAMES]
    toward = [_randn(gen, *t.shape, scale=0.3 if k in ("g", "beta") else 1.0) for k, t in zip(NAMES, rows)]
    weight = s["dy"].double()

    def loss(leaves):
        return (delta_rule(*leaves, state=s["state"], resets=s["resets"])[0].double() * weight).sum()

    leaves = _leaves(s)
    slope = sum(float((g * d).double().sum()) for g, d in zip(torch.autograd.grad(loss(leaves), leaves), toward))
    wide = [ref.f64(t) for t in rows]
    step = 2.0**-14  # 64 bits: what is off is the third derivative, about 100 times the slope, and 2^-28 of it

    def exact(sign):
        moved = [t + sign * step * d.cpu().double() for t, d in zip(wide, toward)]
        return float((_plain(*moved, ref.f64(s["state"]), s["resets"].cpu())[0] * weight.cpu()).sum())

    difference = (exact(1) - exact(-1)) / (2 * step)
    size = sum(float((g * d).double().square().sum()) for g, d in zip(torch.autograd.grad(loss(leaves), leaves), toward)) ** 0.5
    assert abs(difference - slope) < 4 * _roundings(37, 20) * 2.0**-23 * size * 3 + 100 * abs(slope) * 2.0**-28


def test_no_steps_and_no_envs():
    from gbxcule_amd.rl import delta_rule, delta_rule_step

    for steps, envs in ((0, 3), (4, 0)):
        s = _inputs(2, steps, envs, 2, 8, 8)
        leaves = _leaves(s)
        y, last = delta_rule(*leaves, state=s["state"])
        assert y.shape == (steps, envs, 2, 8) and torch.equal(last, s["state"])
        for g, t in zip(torch.autograd.grad(y.sum(), leaves), leaves):
            assert g.shape == t.shape and not g.any()
        y, last = delta_rule(*(s[k] for k in NAMES))
        assert last.shape == (envs, 2, 8, 8) and not last.any()
    empty = torch.zeros(0, 2, 8, 8, device="cuda")
    s = _inputs(2, 1, 0, 2, 8, 8)
    assert delta_rule_step(*(s[k][0] for k in NAMES), state=empty).shape == (0, 2, 8)


def test_some_gradients_alone():
    from gbxcule_amd.rl import delta_rule

    s = _inputs(11, 20, 2, 2, 16, 16)
    every = _leaves(s)
    want = torch.autograd.grad(delta_rule(*every)[0], every, s["dy"])
    for i in range(5):
        leaves = [s[k].detach() for k in NAMES]
        leaves[i].requires_grad_()
        (g,) = torch.autograd.grad(delta_rule(*leaves)[0], leaves[i], s["dy"])
        assert torch.equal(g, want[i])


def test_another_stream_and_a_graph():
    from gbxcule_amd.rl import delta_rule, delta_rule_step

    s = _inputs(12, 40, 3, 2, 32, 32, dtype=BF16, resets=0.1)
    rows = [s[k] for k in NAMES]
    want = delta_rule(*rows, state=s["state"], resets=s["resets"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = delta_rule(*rows, state=s["state"], resets=s["resets"])
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    one = [r[0].clone() for r in rows]
    state, other = s["state"].clone(), s["state"].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = delta_rule(*rows, state=s["state"], resets=s["resets"])
        step = delta_rule_step(*one, state=state)
    state.copy_(s["state"])
    for k in range(3):
        rows[2].copy_(_randn(_gen(50 + k), *rows[2].shape, dtype=BF16))
        one[2].copy_(rows[2][0])
        graph.replay()
        torch.cuda.synchronize()
        want = delta_rule(*rows, state=s["state"], resets=s["resets"])
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        assert torch.equal(step, delta_rule_step(*one, state=other)) and torch.equal(state, other)


def test_refusals():
    import torch.autograd.forward_ad as fwad

    from gbxcule_amd.rl import delta_rule, delta_rule_step

    s = _inputs(1, 4, 2, 4, 8, 8, share=2)
    q, k, v, g, beta = (s[n] for n in NAMES)
    state = s["state"]
    one = [t[0] for t in (q, k, v, g, beta)]
    for bad in (
        lambda: delta_rule(q.cpu(), k, v, g, beta),
        lambda: delta_rule(q, k, v.cpu(), g, beta),
        lambda: delta_rule(q, k, v.double(), g, beta),
        lambda: delta_rule(q.half(), k, v, g, beta),
        lambda: delta_rule(q, k[..., :7], v, g, beta),
        lambda: delta_rule(q[:, :, :1].expand(4, 2, 3, 8), k, v, g, beta),
        lambda: delta_rule(q[:3], k, v, g, beta),
        lambda: delta_rule(q, k, v, g[..., :3], beta),
        lambda: delta_rule(q, k, v, g, beta.int()),
        lambda: delta_rule(q, k, v, g, beta.cpu()),
        lambda: delta_rule(q[0], k, v, g, beta),
        lambda: delta_rule(q, k, v[0], g, beta),
        lambda: delta_rule(q, k, v, g, beta, state=state[:1]),
        lambda: delta_rule(q, k, v, g, beta, state=state.half()),
        lambda: delta_rule(q, k, v, g, beta, state=state.clone().requires_grad_()),
        lambda: delta_rule(q, k, v, g, beta, resets=torch.zeros(4, 3, dtype=torch.bool, device="cuda")),
        lambda: delta_rule(q, k, v, g, beta, resets=torch.zeros(4, 2, device="cuda")),
        lambda: delta_rule(q.repeat(1, 1, 1, 17), k.repeat(1, 1, 1, 17), v, g, beta),  # 136 keys
        lambda: delta_rule(q, k, v.repeat(1, 1, 1, 17), g, beta),
        lambda: delta_rule(q[..., :0], k[..., :0], v, g, beta),
        lambda: delta_rule_step(*one, state=state.transpose(-1, -2)),
        lambda: delta_rule_step(*one, state=state.half()),
        lambda: delta_rule_step(q, k, v, g, beta, state=state),
    ):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        delta_rule_step(*one)  # the state is what it moves
    with pytest.raises(RuntimeError, match="no gradient"):
        delta_rule_step(one[0].clone().requires_grad_(), *one[1:], state=state)
    leaf = v.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(delta_rule(q, k, leaf, g, beta)[0].sum(), leaf, create_graph=True)
    with fwad.dual_level(), pytest.raises(NotImplementedError):
        delta_rule(q, k, fwad.make_dual(v, torch.ones_like(v)), g, beta)
    version = state._version
    delta_rule_step(*one, state=state)
    assert state._version == version + 1


def _behind(s, at, leaves, got, normalize=True):
    """Gradients of the steps from `at` on, where every env begins an episode, against those of these steps alone."""
    rest = {k: s[k][at:] for k in (*NAMES, "dy")}
    wide = [ref.f64(rest[k]).requires_grad_() for k in NAMES]
    want, _ = _plain(*wide, None, None, normalize)
    n = _roundings(len(rest["q"]), s["q"].shape[3])
    for a, b, leaf, name in zip(got, torch.autograd.grad(want, wide, ref.f64(rest["dy"])), leaves, NAMES):
        assert torch.isfinite(a[at:]).all(), name
        terms = _terms(wide, {**rest, "state": None, "resets": None}, None)[name] if normalize and name in "qk" else 0.0
        # what is redone span by span computes u anew, another order of the same sums
        _check_terms(a[at:], b, 2 * 4 * n + s["v"].shape[3], terms, f"gradient of {name}")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("keys, values", [(64, 64), (24, 40)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("closed", [False, True])
def test_a_state_that_an_episode_at_the_first_step_leaves_behind(dtype, keys, values, bad, closed):
    """Fresh memory as a state, with an episode that begins, or a gate that closes, at step 0: no gradient sees it."""
    from gbxcule_amd.rl import delta_rule

    s = _inputs(70, 19, 2, 2, keys, values, dtype=dtype)
    state = s["state"].clone()
    state[1, 0, 3, 5] = bad
    state[0] = bad
    resets = None
    if closed:
        s["g"][0] = -200.0
    else:
        resets = torch.zeros(19, 2, dtype=torch.bool, device="cuda")
        resets[0] = True
    leaves = _leaves(s)
    y, last = delta_rule(*leaves, state=state, resets=resets)
    assert torch.isfinite(y).all() and torch.isfinite(last).all()
    _behind(s, 0, leaves, torch.autograd.grad(y, leaves, s["dy"]))


def test_a_state_that_overflows_right_before_an_episode():
    """The last correction of a chunk is finite and takes the state past the largest number; an episode begins with the next chunk."""
    from gbxcule_amd.rl import delta_rule

    s = _inputs(71, 36, 1, 1, 16, 16, normalize=False)
    for k in ("q", "k", "v", "g", "beta", "dy"):
        s[k][:16] = 0.0
    s["k"][15, ..., :2], s["beta"][15], s["v"][15] = 0.5, 1.0, 1e38
    state = torch.zeros(1, 1, 16, 16, device="cuda")
    state[..., 0, :], state[..., 1, :] = 3.3e38, -3.3e38  # of which the key reads nothing, and adds 0.5e38 to the one
    resets = torch.zeros(36, 1, dtype=torch.bool, device="cuda")
    resets[16] = True
    leaves = _leaves(s)
    y, last = delta_rule(*leaves, state=state, resets=resets, normalize=False)
    assert torch.isfinite(y[16:]).all() and torch.isfinite(last).all()
    _behind(s, 16, leaves, torch.autograd.grad(y, leaves, s["dy"]), False)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("keys, values", [(64, 64), (24, 40)])
@pytest.mark.parametrize("at", [0, 16])
@pytest.mark.parametrize("bad", [math.nan, math.inf, 3e38])
def test_a_correction_right_before_an_episode(dtype, keys, values, at, bad):
    """The correction of a chunk's first step is in no other's: one that is not finite, or is only with what it
    is made of, leaves the system as it is, and no gradient of the episode that begins behind it sees it."""
    from gbxcule_amd.rl import delta_rule

    s = _inputs(72, 36, 2, 2, keys, values, dtype=dtype)
    s["beta"][at] = bad
    s["v"][at, ..., ::2], s["v"][at, ..., 1::2] = 100.0, -100.0
    resets = torch.zeros(36, 2, dtype=torch.bool, device="cuda")
    resets[at + 1] = True
    leaves = _leaves(s)
    y, last = delta_rule(*leaves, state=s["state"], resets=resets)
    assert torch.isfinite(y[at + 1 :]).all() and torch.isfinite(last).all()
    _behind(s, at + 1, leaves, torch.autograd.grad(y, leaves, s["dy"]))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("keys, values", [(64, 64), (24, 40)])
@pytest.mark.parametrize("at", [1, 7, 16, 21])
@pytest.mark.parametrize("big", [1e19, 1e30, 3e38])
def test_large_values_before_an_episode(dtype, keys, values, at, big):
    """Memory that nothing has written holds such numbers as often as ones that are not finite: products of
    them overflow, and zero, which is what an episode's start leaves of them, times infinity is no zero."""
    from gbxcule_amd.rl import delta_rule

    big = min(big, torch.finfo(dtype).max)
    for which in ("q", "k", "v", "beta", "g", "state", "q k", "k v", "q k v g beta state"):
        for normalize in (True, False):
            s = _inputs(73, 40, 2, 2, keys, values, dtype=dtype, normalize=normalize)
            gen = _gen(74)
            for name in which.split():
                t = s[name] if name == "state" else s[name][:at]
                t.copy_(torch.where(_rand(gen, *t.shape) < 0.3, big * torch.sign(_randn(gen, *t.shape)), t.float()))
            resets = torch.zeros(40, 2, dtype=torch.bool, device="cuda")
            resets[at] = True
            leaves = _leaves(s)
            y, last = delta_rule(*leaves, state=s["state"], resets=resets, normalize=normalize)
            want, want_last = _plain(*(ref.f64(s[k][at:]) for k in NAMES), None, None, normalize)
            ref.check(y[at:], want, _roundings(40, keys), f"y after {which}")
            ref.check(last, want_last, _roundings(40, keys), f"state after {which}")
            _behind(s, at, leaves, torch.autograd.grad(y, leaves, s["dy"]), normalize)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("steps, at, keys, values", [(40, 1, 64, 64), (40, 16, 24, 40), (40, 23, 64, 64), (33, 32, 128, 48), (520, 300, 32, 24)])
def test_memory_that_nothing_has_written_before_an_episode(dtype, steps, at, keys, values):
    """Any bits at all, in everything from before it."""
    from gbxcule_amd.rl import delta_rule

    for seed in range(6):
        s = _inputs(75 + seed, steps, 1, 2, keys, values, dtype=dtype)
        gen = _gen(90 + seed)
        for name in (*NAMES, "state"):
            t = s[name] if name == "state" else s[name][:at]
            word = torch.int32 if t.dtype is F32 else torch.int16
            bits = torch.randint(-(2**31), 2**31, t.shape, device="cuda", generator=gen)
            t.copy_(bits.to(word).view(t.dtype))
        resets = torch.zeros(steps, 1, dtype=torch.bool, device="cuda")
        resets[at] = True
        leaves = _leaves(s)
        y, last = delta_rule(*leaves, state=s["state"], resets=resets)
        want, want_last = _plain(*(ref.f64(s[k][at:]) for k in NAMES), None, None)
        ref.check(y[at:], want, _roundings(steps, keys), "y")
        ref.check(last, want_last, _roundings(steps, keys), "state")
        _behind(s, at, leaves, torch.autograd.grad(y, leaves, s["dy"]))


@pytest.mark.parametrize("keys", [16, 33, 64, 128])
def test_products_of_keys_in_float16(keys):
    """1 + 2^-8 and its products have no more digits than 32-bit sums hold in any order, so that all
    that is off in a state is its few roundings, of 2^-24 each: two of a length's root and sum, one of u, two of what
    scales it, one of its parts and up to six of the terms added. A bfloat16 holds the 1, and the square of what it
    leaves is 2^-16 of the product: half of that, of a length's root, would be 128 of these roundings."""
    from gbxcule_amd.rl import delta_rule, delta_rule_step

    gen = _gen(80)
    sign = torch.where(_rand(gen, 1, 3, 2, keys) < 0.5, -1.0, 1.0)
    q = k = (sign * (1.0 + 2.0**-8)).to(F16)
    v, g, beta = _randn(gen, 1, 3, 2, 40, dtype=F16), torch.zeros(1, 3, 2, device="cuda"), torch.full((1, 3, 2), 0.75, device="cuda")
    _, last = delta_rule(q, k, v, g, beta)
    _, want = _plain(*(ref.f64(t) for t in (q, k, v, g, beta)), None, None)
    ref.check(last, want, 8, "state of unit keys")
    state = torch.zeros_like(last)
    delta_rule_step(*(t[0] for t in (q, k, v, g, beta)), state=state)
    ref.check(state, want, 8, "state of a single step")
    # keys of their own length, the same one at two steps, the second of which corrects the first: the product is in
    # what is recalled, and both steps' roundings in the state, which is half of what they are of
    k2 = torch.cat([k, k]) * 2.0**-3 if keys == 64 else torch.cat([k, k]) * 2.0**-4
    rows = [k2, k2, torch.cat([v, torch.zeros_like(v)]), torch.cat([g, g]), torch.cat([beta, beta])]
    _, last = delta_rule(*rows, normalize=False)
    _, want = _plain(*(ref.f64(t) for t in rows), None, None, False)
    ref.check(last, want, 32, "state of plain keys")
