"""AdamW as torch's optimizers are used beside ``step``: copied, pickled,
loaded with hooks, over parameters of several types and in several groups."""

from __future__ import annotations

import copy
import io
import pickle

import pytest
import torch

from . import _policy_ref as ref
from .conftest import require_gpu
from .test_gpu_adamw import BF16, F16, F32, _formula, _params

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu():
    require_gpu()


def _gradients(params, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    for p in params:
        p.grad = torch.randn(p.shape, device="cuda", generator=gen).to(p.dtype)


def _two_groups(bits, seed=4):
    from gbxcule_amd.rl import AdamW

    gen = torch.Generator(device="cuda").manual_seed(seed)
    params = _params(gen, F32) + _params(gen, BF16, [(300,), (7, 9)])
    groups = [{"params": params[:5], "lr": 0.01}, {"params": params[5:], "weight_decay": 0.2}]
    return params, AdamW(groups, lr=0.003, betas=(0.8, 0.95), state_bits=bits, seed=seed)


def _all(opt):
    return [p for g in opt.param_groups for p in g["params"]]


def _pickled(opt):
    return pickle.loads(pickle.dumps(opt))


def _saved(opt):
    file = io.BytesIO()
    torch.save(opt, file)
    file.seek(0)
    return torch.load(file, weights_only=False)


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("way", [copy.deepcopy, _pickled, _saved])
def test_a_copy_steps_as_the_original_does(bits, way):
    params, one = _two_groups(bits)
    for t in range(3):
        _gradients(params, t)
        one.step()
    two = way(one)
    assert type(two) is type(one) and two.state_bits == bits and two.seed == 4
    assert all(p is not q and torch.equal(p, q) for p, q in zip(_all(one), _all(two)))
    for g in range(2):
        for (k, a), b in zip(one.flat_state(g).items(), two.flat_state(g).values()):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)) and a.data_ptr() != b.data_ptr(), k
    before = [p.detach().clone() for p in params]
    _gradients(_all(two), 3)
    two.step()
    assert all(torch.equal(p, q) for p, q in zip(params, before))  # the original's are its own
    assert all(s["step"] == 3 for s in one.state.values()) and all(s["step"] == 4 for s in two.state.values())
    _gradients(params, 3)
    one.step()
    for p, q in zip(_all(one), _all(two)):
        assert torch.equal(p, q)
        for k, v in one.state[p].items():
            mine = two.state[q][k]
            assert v == mine if k == "step" else torch.equal(v.float(), mine.float()), k
    two.load_state_dict(one.state_dict())
    two.add_param_group({"params": [torch.nn.Parameter(torch.ones(5, device="cuda"))]})
    _gradients(_all(two), 4)
    two.step()


def test_a_shallow_copy_leaves_the_original_alone():
    params, one = _two_groups(32)
    _gradients(params, 0)
    one.step()
    copy.copy(one)
    moments = [one.state[p]["exp_avg"].clone() for p in params]
    one.step()
    for p, m in zip(params, moments):
        if p.numel():
            assert not torch.equal(one.state[p]["exp_avg"], m)


def test_load_hooks_run():
    params, one = _two_groups(32)
    _gradients(params, 0)
    one.step()
    kept = one.state_dict()
    seen = []

    def faster(opt, state):
        seen.append(("pre", opt is one, state is not kept))
        return {**state, "param_groups": [{**g, "lr": 9.0} for g in state["param_groups"]]}

    one.register_load_state_dict_pre_hook(faster)
    one.register_load_state_dict_post_hook(lambda opt: seen.append(("post", opt is one, opt.param_groups[0]["lr"])))
    one.load_state_dict(kept)
    assert seen == [("pre", True, True), ("post", True, 9.0)] and kept["param_groups"][0]["lr"] == 0.01


def test_a_state_with_something_missing_is_refused_whole():
    params, one = _two_groups(8)
    _gradients(params, 0)
    one.step()
    kept = copy.deepcopy(one.state_dict())
    _gradients(params, 1)
    one.step()
    now = {k: v.float().clone() for k, v in one.flat_state().items()}
    for spoil in (lambda s: s["state"].pop(3), lambda s: s["state"][2].pop("exp_avg_scale"), lambda s: s["state"][2].pop("step"), lambda s: s.pop("seed"),
                  lambda s: s["state"][12].update(exp_avg=torch.zeros(2)), lambda s: s.pop("state"), lambda s: s.pop("param_groups")):  # fmt: skip
        bad = copy.deepcopy(kept)
        spoil(bad)
        with pytest.raises(ValueError):
            one.load_state_dict(bad)
        assert all(s["step"] == 2 for s in one.state.values())
        assert all(torch.equal(v.float(), now[k]) for k, v in one.flat_state().items())
    one.load_state_dict(kept)
    assert all(s["step"] == 1 for s in one.state.values())


def test_groups_round_apart():
    """Equal parameters and gradients in three groups: the moments' roundings
    fall by odds of their own, and about a third of 4,096 elements turn another way."""
    from gbxcule_amd.rl import AdamW

    gen = torch.Generator(device="cuda").manual_seed(5)
    params = [torch.nn.Parameter(torch.zeros(4096, device="cuda")) for _ in range(3)]
    opt = AdamW([{"params": [p]} for p in params], state_bits=8)
    grad = torch.randn(4096, device="cuda", generator=gen)
    for p in params:
        p.grad = grad.clone()
    opt.step()
    for key in ("exp_avg", "exp_avg_sq"):
        a, b, c = (opt.flat_state(g)[key].float() for g in range(3))
        for u, v in ((a, b), (a, c), (b, c)):
            assert 0.1 < float((u != v).float().mean()) < 0.9, key


def test_parameters_of_several_types():
    """As a policy of 16-bit matrices and 32-bit vectors has them."""
    from gbxcule_amd.rl import AdamW

    gen = torch.Generator(device="cuda").manual_seed(7)
    kinds = [F32, BF16, F16] * 4
    params = [_params(gen, kind, [shape])[0] for kind, shape in zip(kinds, [(3,), (40, 30), (257,), (256,), (1,), (5, 5), (0,), (70, 7), (9,), (4097,), (2,), (64,)])]
    opt = AdamW(params, lr=0.01, betas=(0.8, 0.99), eps=1e-6, weight_decay=0.1)
    state = [[torch.zeros(p.shape, dtype=torch.float64) for _ in range(2)] for p in params]
    for t in range(1, 4):
        before = [p.detach().cpu().double() for p in params]
        _gradients(params, t)
        opt.step()
        for i, p in enumerate(params):
            want, *state[i] = _formula(before[i], p.grad.cpu().double(), *state[i], t, 0.01, 0.8, 0.99, 1e-6, 0.1)
            ref.check(p, want, 32, f"parameter {i} after step {t}")
            ref.check(opt.state[p]["exp_avg"], state[i][0], 8 * t, f"first moment {i}")
            ref.check(opt.state[p]["exp_avg_sq"], state[i][1], 8 * t, f"second moment {i}")
            assert opt.state[p]["step"] == t
