"""AdamW over many tensors against the formula in 64 bits, its 8-bit states
against the same rounding written in torch, and what keeps them moving."""

from __future__ import annotations

import math

import pytest
import torch

from . import _policy_ref as ref
from .conftest import require_gpu

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
SHAPES = [(1,), (3,), (255,), (256,), (257,), (33, 65), (0,), (4096,), (4097,), (2, 3, 5), (70, 300)]


@pytest.fixture(autouse=True)
def _gpu():
    require_gpu()


def _params(gen, dtype, shapes=SHAPES):
    return [torch.nn.Parameter((torch.randn(s, device="cuda", generator=gen)).to(dtype)) for s in shapes]


def _formula(p, g, m, v, t, lr, b1, b2, eps, wd):
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    return p * (1 - lr * wd) - lr * (m / (1 - b1**t)) / (torch.sqrt(v / (1 - b2**t)) + eps), m, v


@pytest.mark.parametrize("dtype, grad_dtype", [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16)])
def test_32_bit_states(dtype, grad_dtype):
    from gbxcule_amd.rl import AdamW

    gen = torch.Generator(device="cuda").manual_seed(1)
    params = _params(gen, dtype)
    opt = AdamW(params, lr=0.01, betas=(0.8, 0.99), eps=1e-6, weight_decay=0.1)
    state = [[torch.zeros(p.shape, dtype=torch.float64) for _ in range(2)] for p in params]
    clip = torch.tensor([0.5], device="cuda")
    for t in range(1, 5):
        before = [p.detach().cpu().double() for p in params]
        for p in params:
            grad = torch.randn(p.shape, device="cuda", generator=gen).to(grad_dtype)
            p.grad = grad if dtype is grad_dtype else None
            if dtype is not grad_dtype:  # torch refuses to assign another type: set it as hooks of mixed precision do
                p.grad_dtype = grad_dtype
                p.grad = grad
        opt.step(grad_scale=clip if t == 3 else None)
        for i, p in enumerate(params):
            g = p.grad.cpu().double() * (0.5 if t == 3 else 1.0)
            want, *state[i] = _formula(before[i], g, *state[i], t, 0.01, 0.8, 0.99, 1e-6, 0.1)
            ref.check(p, want, 32, f"parameter {i} after step {t}")
            ref.check(opt.state[p]["exp_avg"], state[i][0], 8 * t, f"first moment {i}")
            ref.check(opt.state[p]["exp_avg_sq"], state[i][1], 8 * t, f"second moment {i}")
            assert opt.state[p]["step"] == t


def _round_8(t, noise16, mantissa, least, kind):
    cut = 23 - mantissa
    bits = t.abs().view(torch.int32)
    normal = ((bits + (noise16 << (cut - 16))) & ~((1 << cut) - 1)).view(torch.float32)
    quantum = least / (1 << mantissa)
    n = t.abs() / quantum
    small = (n.floor() + (n - n.floor() + noise16.float() * 2.0**-16).floor()) * quantum
    return torch.copysign(torch.where(t.abs() < least, small, normal), t).to(kind)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_8_bit_states(dtype):
    """The same rounding of the same numbers, which differ by a few units in the
    last place of 32 bits: the states agree but for values that near to where
    they turn, fewer than 1 in 1,000."""
    from gbxcule_amd.rl import AdamW

    gen = torch.Generator(device="cuda").manual_seed(2)
    params = _params(gen, dtype)
    lr, b1, b2, eps, wd, seed = 1e-2, 0.9, 0.999, 1e-8, 0.01, 77
    opt = AdamW(params, lr=lr, betas=(b1, b2), eps=eps, weight_decay=wd, state_bits=8, seed=seed)
    for t in range(1, 4):
        flat = {k: v.cpu().clone() for k, v in opt.flat_state().items()}
        before = [p.detach().cpu().float() for p in params]
        for p in params:
            spread = torch.exp(3 * torch.randn(p.shape, device="cuda", generator=gen))
            p.grad = (torch.randn(p.shape, device="cuda", generator=gen) * spread * 1e-3).to(dtype)
        opt.step()
        after = {k: v.cpu() for k, v in opt.flat_state().items()}
        m = (flat["exp_avg"].float().view(-1, 256) * flat["exp_avg_scale"][:, None]).view(-1)
        v = (flat["exp_avg_sq"].float().view(-1, 256) * flat["exp_avg_sq_scale"][:, None]).view(-1)
        g, at = torch.zeros_like(m), 0
        for p in params:
            g[at : at + p.numel()] = p.grad.cpu().float().reshape(-1)
            at += -(-p.numel() // 256) * 256
        assert at == g.numel()
        m, v = m * b1 + g * (1 - b1), v * b2 + g * g * (1 - b2)
        update = (m * (lr / (1 - b1**t))) / (torch.sqrt(v) * (1 / math.sqrt(1 - b2**t)) + eps)
        at = 0
        for i, p in enumerate(params):
            want = before[i].double() * (1 - lr * wd) - update[at : at + p.numel()].double().view(p.shape)
            ref.check(p, want, 8, f"parameter {i} after step {t}")
            at += -(-p.numel() // 256) * 256
        noise = ref.noise(torch.arange(g.numel()), (seed + t * 0x9E3779B9) & 0xFFFFFFFF)
        for key, x, top, part, fmt in (("exp_avg", m, 448.0, noise & 0xFFFF, (3, 2.0**-6, torch.float8_e4m3fn)),
                                       ("exp_avg_sq", v, 57344.0, noise >> 16, (2, 2.0**-14, torch.float8_e5m2))):  # fmt: skip
            most = x.view(-1, 256).abs().amax(1).clamp_min(1e-30)
            ref.check(after[key + "_scale"], most / top, 4, key + "_scale")
            scaled = (x.view(-1, 256) * (top / most)[:, None]).clamp(-top, top).view(-1)
            q = _round_8(scaled, part.int(), *fmt)
            if key == "exp_avg_sq":
                q = torch.where(scaled > 0, q.float().clamp_min(2.0**-16), 0.0).to(q.dtype)
            differ = q.float() != after[key].float()
            assert float(differ.float().mean()) < 1e-3, key
            # one step of the format at most where they differ
            assert bool(((q.float() - after[key].float()).abs() <= scaled.abs() * 0.26 + 2.0**-8).all())


def test_8_bit_second_moment_follows_a_change():
    """A gradient that falls to a tenth: the second moment's mean over many
    elements follows b2^t as in 32 bits, although one step changes an element
    by a tenth of a per cent.  Rounding noise of one element is 2^-3 of its
    value at most a step; over 65,536 elements and 300 steps (the mean forgets
    with b2) the mean's error is below 2^-3 * sqrt(300 / 65536) = 0.9%.  The block's scale
    moves with its largest element."""
    from gbxcule_amd.rl import AdamW

    p = torch.nn.Parameter(torch.zeros(65_536, device="cuda"))
    opt = AdamW([p], lr=0.0, betas=(0.9, 0.99), weight_decay=0.0, state_bits=8, seed=3)
    want = 0.0
    gen = torch.Generator(device="cuda").manual_seed(4)
    size = 0.5 + torch.rand(p.shape, device="cuda", generator=gen)
    for t in range(300):
        scale = 1.0 if t < 150 else 0.1
        p.grad = size * scale
        opt.step()
        want = 0.99 * want + 0.01 * scale**2
    flat = opt.flat_state()
    v = flat["exp_avg_sq"].float().view(-1, 256) * flat["exp_avg_sq_scale"][:, None]
    got = float((v.view(-1) / size**2).mean())
    assert abs(got / want - 1) < 0.03, (got, want)
    m = flat["exp_avg"].float().view(-1, 256) * flat["exp_avg_scale"][:, None]
    assert abs(float((m.view(-1) / size).mean()) / 0.1 - 1) < 0.01


def test_zero_and_bad_gradients_stay_in_their_block():
    from gbxcule_amd.rl import AdamW

    for bits in (8, 32):
        p = torch.nn.Parameter(torch.ones(1024, device="cuda"))
        opt = AdamW([p], lr=0.1, weight_decay=0.0, state_bits=bits)
        p.grad = torch.zeros_like(p)
        opt.step()
        assert torch.equal(p.detach(), torch.ones_like(p))  # 0 / (0 + eps)
        p.grad = torch.ones_like(p)
        p.grad[300] = float("nan")
        opt.step()
        bad = torch.isnan(p.detach())
        assert bad[300] and int(bad.sum()) == 1
        p.grad = torch.ones_like(p)
        opt.step()
        bad = torch.isnan(p.detach())
        assert bad[300] and not bad[:256].any() and not bad[512:].any()


def test_many_tensors_groups_and_missing_gradients():
    """More tensors than one launch takes, two groups, parameters without a
    gradient and with different counts of steps, against torch's AdamW."""
    from gbxcule_amd.rl import AdamW

    gen = torch.Generator(device="cuda").manual_seed(6)
    mine = _params(gen, F32, [(k % 37 + 1, 13) for k in range(333)])
    theirs = [torch.nn.Parameter(p.detach().clone().double()) for p in mine]
    groups = lambda ps: [{"params": ps[:100], "lr": 0.01}, {"params": ps[100:], "weight_decay": 0.3}]  # noqa: E731
    a, b = AdamW(groups(mine), lr=0.002), torch.optim.AdamW(groups(theirs), lr=0.002)
    for t in range(4):
        for k, (p, q) in enumerate(zip(mine, theirs)):
            p.grad = q.grad = None
            if (k + t) % 5:
                g = torch.randn(p.shape, device="cuda", generator=gen)
                p.grad, q.grad = g, g.double()
        versions = [p._version for p in mine]
        a.step()
        b.step()
        assert all(p._version > v for p, v in zip(mine, versions) if p.grad is not None)
        for p, q in zip(mine, theirs):
            ref.check(p, q, 64)
    a.zero_grad()
    a.step()  # nothing to do


def test_strided_gradients_and_scheduler():
    from gbxcule_amd.rl import AdamW

    p = torch.nn.Parameter(torch.zeros(40, 30, device="cuda"))
    opt = AdamW([p], lr=1.0, weight_decay=0.0)
    p.grad = torch.randn(30, 40, device="cuda").t()
    opt.step()
    # the first step moves by lr * g / (|g| + eps)
    g = p.grad.cpu().double()
    ref.check(p, -g / (g.abs() + 1e-8), 64)
    sched = torch.optim.lr_scheduler.LambdaLR(opt, lambda k: 0.0)
    before = p.detach().clone()
    opt.step()
    assert torch.equal(before, p.detach()) and sched.get_last_lr() == [0.0]


@pytest.mark.parametrize("bits", [8, 32])
def test_state_dict_round_trip(bits):
    from gbxcule_amd.rl import AdamW

    def run(opt, params, steps, first):
        for t in range(first, first + steps):
            gen = torch.Generator(device="cuda").manual_seed(100 + t)
            for p in params:
                p.grad = torch.randn(p.shape, device="cuda", generator=gen)
            opt.step()

    gen = torch.Generator(device="cuda").manual_seed(8)
    a = _params(gen, F32)
    one = AdamW(a, state_bits=bits, seed=9)
    run(one, a, 3, 0)
    kept, values = one.state_dict(), [p.detach().clone() for p in a]
    kept = {k: ({i: {n: (t.clone() if torch.is_tensor(t) else t) for n, t in s.items()} for i, s in v.items()} if k == "state" else v)
            for k, v in kept.items()}  # fmt: skip
    run(one, a, 2, 3)
    b = [torch.nn.Parameter(v) for v in values]
    two = AdamW(b, lr=5.0, state_bits=bits)
    two.load_state_dict(kept)
    assert two.param_groups[0]["lr"] == 1e-3 and two.seed == 9
    run(two, b, 2, 3)
    for p, q in zip(a, b):
        assert torch.equal(p.detach(), q.detach())
    three = AdamW([torch.nn.Parameter(v) for v in values], state_bits=40 - bits)
    with pytest.raises(ValueError):
        three.load_state_dict(kept)


def test_refusals():
    from gbxcule_amd.rl import AdamW

    p = torch.nn.Parameter(torch.zeros(8, 4, device="cuda"))
    for bad in (dict(state_bits=16), dict(lr=-1.0), dict(eps=0.0), dict(betas=(1.0, 0.9)), dict(weight_decay=-0.1)):
        with pytest.raises(ValueError):
            AdamW([p], **bad)
    for q in (torch.zeros(3), torch.zeros(3, device="cuda", dtype=torch.float64), torch.zeros(4, 4, device="cuda").t()[:2]):
        with pytest.raises(ValueError):
            AdamW([torch.nn.Parameter(q)])
    opt = AdamW([p])
    p.grad = torch.zeros_like(p)
    with pytest.raises(ValueError):
        opt.step(grad_scale=torch.zeros(2, device="cuda"))
    with pytest.raises(ValueError):
        opt.load_flat_state(1, {})
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(graph):
            opt.step()


def test_hooks_and_profiler():
    """Hooks on the step run once, before and after it, whether the optimizer's
    own or for all optimizers; a profiler sees the step; a scheduler counts it."""
    from torch.optim.optimizer import register_optimizer_step_post_hook, register_optimizer_step_pre_hook

    from gbxcule_amd.rl import AdamW

    p = torch.nn.Parameter(torch.ones(10, device="cuda"))
    opt = AdamW([p], lr=0.5)
    p.grad = torch.ones_like(p)
    seen = []
    note = lambda name: lambda o, args, kwargs: seen.append((name, o is opt, opt.state[p]["step"]))  # noqa: E731
    opt.step()
    handles = [opt.register_step_pre_hook(note("pre"))]
    opt.step()
    assert seen == [("pre", True, 1)]
    handles.append(opt.register_step_post_hook(note("post")))
    opt.step()
    assert seen[1:] == [("pre", True, 2), ("post", True, 3)]
    for h in handles:
        h.remove()
    seen.clear()
    handles = [register_optimizer_step_pre_hook(note("all pre")), register_optimizer_step_post_hook(note("all post"))]
    try:
        opt.step(lambda: seen.append("closure"))
    finally:
        for h in handles:
            h.remove()
    assert seen == [("all pre", True, 3), "closure", ("all post", True, 4)]
    opt.step()
    assert len(seen) == 3 and opt.state[p]["step"] == 5
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as prof:
        opt.step()
    assert any(e.key.startswith("Optimizer.step#AdamW") for e in prof.key_averages())
    schedule = torch.optim.lr_scheduler.StepLR(opt, 1, gamma=0.1)
    opt.step()
    schedule.step()
    assert opt.state[p]["step"] == 7 and opt.param_groups[0]["lr"] == pytest.approx(0.05)
