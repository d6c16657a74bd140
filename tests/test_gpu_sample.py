"""Sampling against a plain 64-bit form that sorts each row: action counts around
every variant's, types, options as numbers and one a row, equals, actions that are
not allowed, infinities and NaN, random numbers at the ends, shares of a spread of
random numbers, streams, graphs, and refusals."""

from __future__ import annotations

import itertools
import math

import pytest
import torch

from .conftest import require_gpu

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _gpu():
    require_gpu()


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _plain_row(x, u, heat, k, p, least):
    """(action, logp) of one row: x float64 on the CPU, the rest numbers."""
    x = torch.where(torch.isnan(x), -math.inf, x)
    most = float(x.max())
    if most == -math.inf:
        return -1, math.nan
    if not heat > 0 or not p > 0 or not least <= 1:
        k, p, least = 1, 1.0, 0.0
    if not heat > 0 or most == math.inf:
        w = (x == most).double()
    else:
        w = torch.where(x == -math.inf, 0.0, torch.exp((x - most) / heat))
    order = torch.sort(x, descending=True, stable=True).indices
    if k > 0:
        order = order[:k]
    ranked = w[order]
    before = ranked.cumsum(0) - ranked
    before[0] = 0.0
    stays = ranked >= least
    if p < 1:
        stays &= before < p * float(ranked.sum())
    stays[0] = True
    kept = torch.zeros_like(w)
    kept[order[stays]] = ranked[stays]
    run = kept.cumsum(0)
    past = torch.nonzero((run > u * run[-1]) & (kept > 0)).flatten()
    action = int(past[0]) if len(past) else int(torch.nonzero(kept > 0).flatten()[-1])
    return action, math.log(float(kept[action] / run[-1]))


def _check(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    from gbxcule_amd.rl import sample_actions

    options = {"temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p}
    action, logp = sample_actions(logits, uniform, **options)
    assert action.dtype is torch.int32 and logp.dtype is F32 and action.shape == logp.shape == logits.shape[:-1]
    rows = logits.reshape(-1, logits.shape[-1]).cpu().double()
    each = [o.reshape(-1).tolist() if isinstance(o, torch.Tensor) else [o] * len(rows) for o in options.values()]
    for i, (got, lp, u) in enumerate(zip(action.reshape(-1).tolist(), logp.reshape(-1).tolist(), uniform.reshape(-1).tolist())):
        want, want_lp = _plain_row(rows[i], u, *(o[i] for o in each))
        assert got == want, (i, u, [o[i] for o in each], got, want)
        # 64 bits, rounded once
        assert lp == want_lp or (math.isnan(lp) and math.isnan(want_lp)) or abs(lp - want_lp) <= 2.0**-24 * abs(want_lp) + 1e-15, (i, lp, want_lp)
    return action, logp


SIZES = [1, 2, 7, 8, 9, 16, 17, 32, 33, 63, 64, 65, 500, 512, 513, 2048, 2049, 10_000, 16_384, 16_385, 40_001]


@pytest.mark.parametrize("actions", SIZES)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_against_sorting(actions, dtype):
    gen = _gen(actions)
    rows = 97 if actions <= 64 else 11
    scale = 0.3 * 20.0 ** torch.rand(rows, 1, device="cuda", generator=gen)
    logits = (torch.randn(rows, actions, device="cuda", generator=gen) * scale).to(dtype)
    u = torch.rand(rows, device="cuda", generator=gen)
    for options in (
        {},
        {"temperature": 0.7},
        {"top_k": 5},
        {"top_p": 0.9},
        {"min_p": 0.05},
        {"temperature": 1.3, "top_k": 40, "top_p": 0.8, "min_p": 0.02},
        {"top_k": actions // 2 + 1, "top_p": 0.99},
        {"temperature": 0.0},
        {"top_k": 1},
        {"top_p": 1e-9},
        {"min_p": 1.0},
        {"temperature": 1e-30},
        {"temperature": math.inf, "top_p": 0.5},
    ):
        _check(logits, u, **options)


@pytest.mark.parametrize("actions", [6, 50, 300, 3000, 20_000])
def test_options_of_each_row(actions):
    gen = _gen(actions + 1)
    shape = (4, 15)
    logits = torch.randn(*shape, actions, device="cuda", generator=gen) * 3
    logits[torch.rand(*shape, actions, device="cuda", generator=gen) < 0.2] = -math.inf
    pick = lambda values, kind=F32: torch.tensor(values, dtype=kind, device="cuda")[  # noqa: E731
        torch.randint(len(values), shape, device="cuda", generator=gen)]  # fmt: skip
    options = {
        "temperature": pick([0.0, 0.5, 1.0, 2.0, -1.0, math.nan, 1e30]),
        "top_k": pick([-3, 0, 1, 2, 5, 40, 2**31 - 1], torch.int32),
        "top_p": pick([1.0, 0.9, 0.5, 0.1, 0.0, -1.0, 2.0, math.nan]),
        "min_p": pick([0.0, 0.1, 0.5, 1.0, 2.0, -1.0, math.nan]),
    }
    u = torch.rand(shape, device="cuda", generator=gen)
    _check(logits, u, **options)
    for name in options:  # one of them alone
        _check(logits, u, **{name: options[name]})


@pytest.mark.parametrize("actions", [8, 40, 700, 17_000])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_equals(actions, dtype):
    """A policy that has learned nothing: cuts and borders fall exactly between equals."""
    gen = _gen(3)
    rows = 40
    u = torch.arange(rows, device="cuda") / rows
    u[:8] = torch.arange(8, device="cuda") / 8
    logits = torch.zeros(rows, actions, device="cuda", dtype=dtype)
    some = torch.randint(0, 3, (rows, actions), device="cuda", generator=gen).to(dtype)  # three values
    zeros = torch.where(torch.rand(rows, actions, device="cuda", generator=gen) < 0.5, -0.0, 0.0).to(dtype)
    for x in (logits, some, zeros):
        for options in ({}, {"top_k": 3}, {"top_p": 0.5}, {"top_p": 0.25, "top_k": 4}, {"min_p": 1.0}, {"temperature": 0.0}):
            _check(x, u, **options)


@pytest.mark.parametrize("actions", [8, 64, 65, 3000, 20_000])
def test_rows_with_little_to_draw_from(actions):
    gen = _gen(4)
    x = torch.randn(9, actions, device="cuda", generator=gen)
    x[0] = -math.inf
    x[1] = math.nan
    x[2, :-1] = -math.inf
    x[3, 1:] = math.nan
    x[4, 2] = math.inf
    x[5, 1:4] = math.inf
    x[6] = math.inf
    x[7, ::2] = math.nan
    u = torch.rand(9, device="cuda", generator=gen)
    for options in ({}, {"top_k": 2}, {"top_p": 0.6}, {"min_p": 0.5}, {"temperature": 0.0}, {"top_k": 3, "top_p": 0.5, "min_p": 0.1}):
        action, logp = _check(x, u, **options)
        assert action[:2].tolist() == [-1, -1] and torch.isnan(logp[:2]).all()
        assert action[2:4].tolist() == [actions - 1, 0] and not logp[2:4].any()
    # random numbers at and past the ends: the first and the last action that stays
    x = torch.randn(6, actions, device="cuda", generator=gen)
    x[:, 0] = -math.inf
    ends = torch.tensor([0.0, 1.0 - 2.0**-24, 1.0, 2.0, -1.0, math.nan], device="cuda")
    action, _ = _check(x, ends)
    assert action[0] == 1 and action[4] == 1 and action[[1, 2, 3, 5]].tolist() == [actions - 1] * 4


@pytest.mark.parametrize("actions", [5, 64, 900, 5000])
def test_shares(actions):
    """Random numbers spread evenly: each action is drawn as often as its probability says, within one."""
    from gbxcule_amd.rl import sample_actions

    n = 4096
    one = torch.randn(actions, device="cuda", generator=_gen(5)) * 2
    u = (torch.arange(n, device="cuda") + 0.5) / n
    action, logp = sample_actions(one.expand(n, actions), u, temperature=0.9)
    weight = torch.exp((one.double() - one.double().max()) / 0.9)
    share = weight / weight.sum()  # (torch's softmax of long 64-bit rows is off by 1e-6)
    counts = torch.bincount(action.long(), minlength=actions)
    assert float((counts - share * n).abs().max()) <= 1.0
    torch.testing.assert_close(logp.double(), share.log()[action.long()], rtol=2.0**-24, atol=1e-14)


def test_shapes_and_strides():
    from gbxcule_amd.rl import sample_actions

    gen = _gen(6)
    wide = torch.randn(7, 5, 31, device="cuda", generator=gen)
    u = torch.rand(7, 5, device="cuda", generator=gen)
    for x in (wide[..., 3:20], wide[..., ::2], wide[:, :, 1:9], wide.transpose(0, 1).contiguous().transpose(0, 1)):
        _check(x, u)
    _check(wide[:, :1].expand(7, 5, 31), u.t().contiguous().t(), top_k=torch.full((5, 7), 4, dtype=torch.int32, device="cuda").t())
    action, logp = sample_actions(wide[0, 0], u[0, 0])
    assert action.shape == logp.shape == () and action == sample_actions(wide[0], u[0])[0][0]
    action, logp = sample_actions(wide[:0], u[:0])
    assert action.shape == logp.shape == (0, 5)


def test_another_stream_and_a_graph():
    from gbxcule_amd.rl import sample_actions

    gen = _gen(7)
    for actions in (9, 600, 20_000):
        x, u = torch.randn(50, actions, device="cuda", generator=gen), torch.rand(50, device="cuda", generator=gen)
        options = {"top_k": 20, "top_p": 0.9}
        want = sample_actions(x, u, **options)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = sample_actions(x, u, **options)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = sample_actions(x, u, **options)
        for _ in range(3):
            x.copy_(torch.randn(50, actions, device="cuda", generator=gen))
            u.copy_(torch.rand(50, device="cuda", generator=gen))
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, sample_actions(x, u, **options)))


def test_refusals():
    from gbxcule_amd.rl import sample_actions

    x, u = torch.randn(4, 8, device="cuda"), torch.rand(4, device="cuda")
    one = torch.ones(4, device="cuda")
    for bad in (
        lambda: sample_actions(x.cpu(), u),
        lambda: sample_actions(x, u.cpu()),
        lambda: sample_actions(x.double(), u),
        lambda: sample_actions(x, u.double()),
        lambda: sample_actions(x, u[:3]),
        lambda: sample_actions(x[:, :0], u),
        lambda: sample_actions(torch.zeros((), device="cuda"), torch.zeros((), device="cuda")),
        lambda: sample_actions(x, u, temperature=-0.1),
        lambda: sample_actions(x, u, temperature=math.nan),
        lambda: sample_actions(x, u, top_p=0.0),
        lambda: sample_actions(x, u, top_p=math.nan),
        lambda: sample_actions(x, u, min_p=1.5),
        lambda: sample_actions(x, u, temperature=one[:2]),
        lambda: sample_actions(x, u, top_p=one.half()),
        lambda: sample_actions(x, u, top_k=one),
        lambda: sample_actions(x, u, min_p=one.cpu()),
    ):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: sample_actions(x, u, top_k=1.5), lambda: sample_actions(x, u, temperature="hot"), lambda: sample_actions(x, 0.5)):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(RuntimeError, match="no gradient"):
        sample_actions(x.clone().requires_grad_(), u)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_one_action_with_any_options(dtype):
    """It is always drawn, whatever the cuts are: every output is written."""
    from gbxcule_amd import _lib

    lib = _lib.load()
    values = {
        "temperatures": [0.0, -1.0, math.nan, 1e-30, 1.0, math.inf],
        "top_ps": [0.0, -1.0, math.nan, 1e-30, 0.5, 1.0],
        "min_ps": [-1.0, 0.0, 1.0, 1.5, math.inf, math.nan],
    }
    grid = torch.tensor(list(itertools.product(*values.values())), device="cuda")
    rows = len(grid)
    ks = torch.tensor([-1, 0, 1, 2], dtype=torch.int32, device="cuda").repeat(rows)[:rows]
    logits = torch.tensor([0.5, -3.0, math.inf, -math.inf, math.nan], device="cuda").repeat(rows)[:rows].to(dtype)
    uniform = torch.rand(rows, device="cuda", generator=_gen(8))
    action, logp = torch.full((rows,), 77, dtype=torch.int32, device="cuda"), torch.full((rows,), 77.0, device="cuda")
    each = [grid[:, i].contiguous() for i in range(3)]
    given = _lib.SampleIn(rows=rows, actions=1, elem={F32: 0, BF16: 1, F16: 2}[dtype], logits=logits.data_ptr(), stride=1, uniform=uniform.data_ptr(),
                          top_ks=ks.data_ptr(), **{k: t.data_ptr() for k, t in zip(values, each)})  # fmt: skip
    assert lib.gbx_sample_actions(given, action.data_ptr(), logp.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
    allowed = logits > -math.inf  # not NaN either
    assert torch.equal(action, torch.where(allowed, 0, -1).int())
    assert not logp[allowed].any() and torch.isnan(logp[~allowed]).all()
    for name, option in zip(("temperature", "top_p", "min_p"), each):  # one of them alone, by the public name
        _check(logits.unsqueeze(1), uniform, **{name: option})


def test_no_derivative_is_dropped():
    """Tangents and gradients are refused, of the logits and of the options."""
    import torch.autograd.forward_ad as fwad

    from gbxcule_amd.rl import sample_actions

    x, u, one = torch.randn(4, 8, device="cuda"), torch.rand(4, device="cuda"), torch.full((4,), 0.5, device="cuda")
    tensors = {"logits": x, "uniform": u, "temperature": one, "top_p": one, "min_p": one}
    for name in tensors:
        leaf = tensors[name].clone().requires_grad_()
        with pytest.raises(RuntimeError, match="no gradient"):
            sample_actions(**{**tensors, name: leaf})
        with torch.no_grad():
            action, logp = sample_actions(**{**tensors, name: leaf})
        want = sample_actions(**tensors)
        assert torch.equal(action, want[0]) and torch.equal(logp, want[1])
        with fwad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
            sample_actions(**{**tensors, name: fwad.make_dual(tensors[name], torch.ones_like(tensors[name]))})
