"""The operators of a policy that remembers, as timed cases.

A policy that reads rollouts (``gbxcule_amd.rl``) keeps a memory of each env's
episode: a block normalises its input (``rms_norm``), mixes the last few steps
(``causal_conv``), runs a selective state space recurrence over the steps
(``selective_scan``) and learns with ``AdamW``.  Everything is time-major as in
``RolloutBuffer``: ``[steps, envs, channels]``, and ``resets[t, n]`` says that
env ``n`` begins an episode at step ``t``, so several episodes of any length
lie one after the other in a row.

The actor makes one step of all envs at a time, from a handful of envs to 128 K
of them; the learner reads whole rollouts forward and backward; an evaluation
runs one long recorded episode as a prompt.

With ``own`` false, ``run`` computes the operators with elementary torch
operations in 32 bits, rounded once at the end.  With ``own`` true it calls the
framework.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
E4M3_MAX, E5M2_MAX = 448.0, 57344.0
SCALE_FLOOR = 1e-30  # the least absolute maximum that an 8-bit scale is made from
STATE_BLOCK = 256  # elements of an 8-bit optimizer state that share a scale
LR, BETAS, EPS, DECAY, ADAM_SEED = 3e-4, (0.9, 0.999), 1e-8, 0.01, 5
NORM_EPS = 1e-6


def _norm(name, kind, rows, dim, dtype="bf16", residual=True, group=0):
    return {"name": name, "kind": kind, "rows": rows, "dim": dim, "dtype": dtype, "residual": residual, "group": group}


def _conv(name, kind, steps, envs, dim, width=4, dtype="bf16", resets=0.0, bias=True, silu=True):
    return {"name": name, "kind": kind, "steps": steps, "envs": envs, "dim": dim, "width": width, "dtype": dtype,
            "resets": resets, "bias": bias, "silu": silu}  # fmt: skip


def _scan(name, kind, steps, envs, dim, states=16, groups=1, dtype="bf16", resets=0.0, gate=True, skip=True,
          bias=True, softplus=True):  # fmt: skip
    return {"name": name, "kind": kind, "steps": steps, "envs": envs, "dim": dim, "states": states, "groups": groups,
            "dtype": dtype, "resets": resets, "gate": gate, "skip": skip, "bias": bias, "softplus": softplus}  # fmt: skip


def _adamw(name, bits, layers, width, dtype="f32"):
    return {"name": name, "kind": "adamw", "bits": bits, "layers": layers, "width": width, "dtype": dtype}


def listed():
    return [
        # acting with 64 envs: one row an env, launch latency
        _norm("norm_act_64", "norm", 64, 256),
        # a learner's minibatch of 128 steps x 1,024 envs, forward and backward
        _norm("norm_train_131072", "norm_train", 131_072, 512),
        # acting in 8 bits at a ragged env count: a scale for each 128 channels
        _norm("norm_fp8_20011", "norm_fp8", 20_011, 1024, group=128),
        # the learner's convolution over a rollout with an episode end here and there
        _conv("conv_train_128x1024", "conv_train", 128, 1024, 1024, resets=0.01),
        # one step of 16,384 envs
        _conv("conv_step_16384", "conv_step", 1, 16_384, 512, resets=0.01),
        # one step of a handful of envs
        _scan("scan_step_64", "scan_step", 1, 64, 512, resets=0.01),
        # one step of 16,384 envs: half a gigabyte of state read and written
        _scan("scan_step_16384", "scan_step", 1, 16_384, 512, resets=0.01),
        # one recorded episode of 16,384 steps as a prompt: one row, a long axis
        _scan("scan_prompt_16384", "scan", 16_384, 1, 1024),
        # the learner's recurrence over a rollout, forward and backward
        _scan("scan_train_128x1024", "scan_train", 128, 1024, 512, resets=0.01),
        # odd sizes in 32 bits, two groups of B and C
        _scan("scan_train_77x37", "scan_train", 77, 37, 200, states=8, groups=2, dtype="f32", resets=0.05),
        # a small policy's update in 32 bits: 20 tensors, latency
        _adamw("adamw_small_32", 32, 2, 256),
        # a large policy's: 240 tensors in bfloat16, states in 8 bits
        _adamw("adamw_large_8", 8, 24, 1024, "bf16"),
    ]  # fmt: skip


def _log_int(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def _channels(rng, lo, hi):
    """A channel count: mostly one that 16-byte loads take, else any."""
    d = _log_int(rng, lo, hi)
    return max(8, d - d % 8) if rng.random() < 0.6 else d


def draw(rng):
    kind = rng.choice(["norm", "norm_train", "norm_fp8", "conv", "conv_train", "conv_step", "scan", "scan_train",
                       "scan_step", "adamw"])  # fmt: skip
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    resets = rng.choice([0.0, 0.005, 0.05, 1.0])
    if kind.startswith("norm"):
        dim = _channels(rng, 24, 8192)
        rows = _log_int(rng, 1, min(131_072, 131_072 * 512 // dim))
        group = rng.choice([0, 128]) if kind == "norm_fp8" else 0
        return _drawn(_norm("", kind, rows, dim, dtype, rng.random() < 0.7, group))
    if kind.startswith("conv"):
        dim, width = _channels(rng, 16, 2048), rng.choice([2, 3, 4, 4])
        if kind == "conv_step":
            steps, envs = 1, _log_int(rng, 1, 16_384 * 512 // dim)
        else:
            most = 128 * 1024 * 1024 // dim // (1 if dtype != "f32" else 2)
            steps = _log_int(rng, 1, min(16_384, most))
            envs = _log_int(rng, 1, max(1, min(16_384, most // steps)))
        return _drawn(_conv("", kind, steps, envs, dim, width, dtype, resets, rng.random() < 0.8, rng.random() < 0.8))
    if kind.startswith("scan"):
        states = rng.choice([4, 8, 12, 16, 16, 16, 24, 32])
        groups = rng.choice([1, 1, 1, 2, 4])
        dim = groups * max(8, _channels(rng, 32, 1024) // groups)
        flags = [rng.random() < 0.7 for _ in range(4)]
        if kind == "scan_step":
            steps, envs = 1, _log_int(rng, 1, 16_384 * 512 * 16 // (dim * states))
        elif kind == "scan":
            most = 16_384 * 1024 * 16 // (dim * states)
            steps = _log_int(rng, 1, min(16_384, most))
            envs = _log_int(rng, 1, max(1, most // steps))
        else:
            most = 128 * 1024 * 512 * 16 // (dim * states) // 2
            steps = _log_int(rng, 1, min(1024, most))
            envs = _log_int(rng, 1, max(1, min(16_384, most // steps)))
        return _drawn(_scan("", kind, steps, envs, dim, states, groups, dtype, resets, *flags))
    return _drawn(_adamw("", rng.choice([8, 32]), rng.randrange(1, 17), _channels(rng, 40, 1024), dtype))


def _drawn(case):
    return {k: v for k, v in case.items() if k != "name"}


# ------------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 13)


def _randn(gen, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, device="cuda", generator=gen) * scale).to(dtype)


def _resets(gen, case, *shape):
    """Episode starts; None where the program has no episodes to part."""
    return torch.rand(shape, device="cuda", generator=gen) < case["resets"] if case["resets"] > 0 else None


def _norm_inputs(case, seed):
    gen, dtype = _gen(seed), DTYPES[case["dtype"]]
    shape = (case["rows"], case["dim"])
    s = {"x": _randn(gen, *shape, dtype=dtype), "weight": 1.0 + _randn(gen, case["dim"], scale=0.1)}
    # a residual stream has grown over the blocks before
    s["residual"] = _randn(gen, *shape, dtype=dtype, scale=3.0) if case["residual"] else None
    if case["kind"] == "norm_train":
        s["dy"] = _randn(gen, *shape, dtype=dtype)
        s["dsummed"] = _randn(gen, *shape, dtype=dtype) if case["residual"] else None
    return s


def _conv_inputs(case, seed):
    gen, dtype = _gen(seed), DTYPES[case["dtype"]]
    steps, envs, dim, width = (case[k] for k in ("steps", "envs", "dim", "width"))
    shape = (steps, envs, dim)
    # x is the first half of a projection's output: rows are 2 x dim apart
    s = {"x": _randn(gen, *shape[:2], 2 * dim, dtype=dtype)[..., :dim]}
    s["weight"] = _randn(gen, dim, width, scale=width**-0.5)
    s["bias"] = _randn(gen, dim, scale=0.1) if case["bias"] else None
    s["state"] = _randn(gen, envs, width - 1, dim, dtype=dtype)
    s["resets"] = _resets(gen, case, steps, envs)
    if case["kind"] == "conv_train":
        s["dy"] = _randn(gen, *shape, dtype=dtype)
    if case["kind"] == "conv_step":
        s["x"] = s["x"][0]
        s["resets"] = None if s["resets"] is None else s["resets"][0]
    return s


def _scan_inputs(case, seed):
    gen, dtype = _gen(seed), DTYPES[case["dtype"]]
    steps, envs, dim, states, groups = (case[k] for k in ("steps", "envs", "dim", "states", "groups"))
    shape = (steps, envs, dim)
    s = {"x": _randn(gen, *shape, dtype=dtype)}
    # the gate is the second half of the projection that x came from; B and C
    # are parts of one projection's output, after the low-rank part of dt
    s["z"] = _randn(gen, *shape[:2], 2 * dim, dtype=dtype)[..., dim:] if case["gate"] else None
    rank, gs = -(-dim // 16), groups * states
    bc = _randn(gen, steps, envs, rank + 2 * gs, dtype=dtype)
    s["B"] = bc[..., rank : rank + gs].unflatten(-1, (groups, states))
    s["C"] = bc[..., rank + gs :].unflatten(-1, (groups, states))
    # step sizes from 0.001 to 0.1, decay rates of about 1 to `states`
    size = 0.001 * 100.0 ** torch.rand(dim, device="cuda", generator=gen)
    raw = size + torch.log(-torch.expm1(-size)) if case["softplus"] else size  # softplus(raw) = size
    noise = _randn(gen, *shape, scale=0.5 if case["softplus"] else 0.0)
    s["dt_bias"] = raw if case["bias"] else None
    s["dt"] = (noise if case["bias"] else noise + raw).to(dtype)
    rates = torch.arange(1, states + 1, device="cuda", dtype=torch.float32)
    s["A"] = -rates * torch.exp(_randn(gen, dim, states, scale=0.1))
    s["D"] = 1.0 + _randn(gen, dim, scale=0.1) if case["skip"] else None
    s["state"] = _randn(gen, envs, dim, states, scale=0.3)
    s["resets"] = _resets(gen, case, steps, envs)
    if case["kind"] == "scan_train":
        s["dy"] = _randn(gen, *shape, dtype=dtype)
    if case["kind"] == "scan_step":
        for k in ("x", "z", "B", "C", "dt", "resets"):
            s[k] = None if s[k] is None else s[k][0]
    return s


def _adamw_shapes(case):
    """The tensors of a memory policy: per block norm, projections,
    convolution and recurrence."""
    d, rank = case["width"], -(-case["width"] // 16)
    block = [(d,), (4 * d, d), (2 * d, 4), (2 * d,), (rank + 32, 2 * d), (2 * d, rank), (2 * d,), (2 * d, 16), (2 * d,),
             (d, 2 * d)]  # fmt: skip
    return block * case["layers"]


def _adamw_inputs(case, seed):
    gen, dtype = _gen(seed), DTYPES[case["dtype"]]
    shapes = _adamw_shapes(case)
    sizes = [math.prod(sh) for sh in shapes]
    starts, total = [], 0
    for n in sizes:  # every tensor starts at a multiple of the block
        starts.append(total)
        total += -(-n // STATE_BLOCK) * STATE_BLOCK
    live = torch.zeros(total, dtype=torch.bool, device="cuda")
    for a, n in zip(starts, sizes):
        live[a : a + n] = True
    # tensors and channels whose gradients differ by orders of magnitude
    spread = torch.exp(2.0 * torch.randn(total // STATE_BLOCK, 1, device="cuda", generator=gen))
    fill = lambda scale, t: (t.view(-1, STATE_BLOCK) * spread * scale).view(-1) * live  # noqa: E731
    s = {"params": _randn(gen, total, dtype=dtype, scale=0.02) * live}
    s["grads"] = fill(1e-3, _randn(gen, total)).to(dtype)
    m = fill(2e-4, _randn(gen, total))
    v = fill(1e-3, _randn(gen, total)).square()
    s["exp_avg"], s["exp_avg_sq"], s["exp_avg_scale"], s["exp_avg_sq_scale"] = m, v, None, None
    if case["bits"] == 8:
        for k, t, top, kind in (("exp_avg", m, E4M3_MAX, torch.float8_e4m3fn),
                                ("exp_avg_sq", v, E5M2_MAX, torch.float8_e5m2)):  # fmt: skip
            t = t.view(-1, STATE_BLOCK)
            most = t.abs().amax(1, keepdim=True).clamp_min(SCALE_FLOOR)
            s[k] = (t * (top / most)).clamp(-top, top).to(kind).view(-1)
            s[k + "_scale"] = (most / top).view(-1)
    s["views"] = [(a, n, sh) for a, n, sh in zip(starts, sizes, shapes)]
    return s


def _inputs(case, seed):
    kind = case["kind"].split("_")[0]
    return {"norm": _norm_inputs, "conv": _conv_inputs, "scan": _scan_inputs, "adamw": _adamw_inputs}[kind](case, seed)


#: What a training step differentiates.
LEAVES = {
    "norm_train": ("x", "residual", "weight"),
    "conv_train": ("x", "weight", "bias"),
    "scan_train": ("x", "dt", "A", "B", "C", "D", "z", "dt_bias"),
}


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    for k in LEAVES.get(case["kind"], ()):
        s[k] = None if s[k] is None else s[k].detach().requires_grad_()
    if case["kind"] == "adamw":
        s["step"] = 9  # passes that the optimizer has made
        s["tensors"] = []
        for a, n, shape in s["views"]:
            p = s["params"][a : a + n].view(shape)
            p.grad = s["grads"][a : a + n].view(shape)
            s["tensors"].append(p)
        if own:  # the optimizer that a program keeps
            from gbxcule_amd.rl import AdamW

            s["opt"] = AdamW(s["tensors"], lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, state_bits=case["bits"],
                             seed=ADAM_SEED)  # fmt: skip
            s["opt"].load_flat_state(s["step"], {k: s[k] for k in s if k.startswith("exp_avg") and s[k] is not None})
    return s


# --------------------------------------------------------------- plain forms


def _plain_rms_norm(x, weight, residual):
    total = x.float() if residual is None else (x.float() + residual.float()).to(x.dtype).float()
    rstd = torch.rsqrt((total * total).mean(-1, keepdim=True) + NORM_EPS)
    return total * rstd * weight, total


def _plain_fp8(y, group):
    rows, dim = y.shape
    size = group or dim
    full = -(-dim // size) * size
    blocks = torch.nn.functional.pad(y, (0, full - dim)).view(rows, -1, size)
    most = blocks.abs().amax(-1, keepdim=True).clamp_min(SCALE_FLOOR)
    q = (blocks * (E4M3_MAX / most)).to(torch.float8_e4m3fn).view(rows, full)[:, :dim]
    scale = (most / E4M3_MAX).squeeze(-1)
    return q, scale if group else scale[:, 0]


def _plain_conv(x, weight, bias, state, resets, silu):
    """x ``[T, N, D]``.  Tap j reaches j steps back, into ``state`` before the
    first step, and not past the start of an episode."""
    steps, width = x.shape[0], weight.shape[1]
    past = torch.cat([state, x])
    window = past.float()
    if resets is not None:  # episodes counted along the row
        episode = torch.cat([torch.zeros_like(resets[:1], dtype=torch.int32).expand(width - 1, -1), resets.cumsum(0)])
        episode = episode.unsqueeze(-1)
    pre = 0.0 if bias is None else bias
    for j in range(width):
        tap = window[width - 1 - j : width - 1 - j + steps]
        if resets is not None and j:
            tap = torch.where(episode[width - 1 - j : width - 1 - j + steps] == episode[width - 1 :], tap, 0.0)
        pre = pre + tap * weight[:, width - 1 - j]
    y = pre * torch.sigmoid(pre) if silu else pre
    kept = past[steps:]
    if resets is not None:
        kept = torch.where(episode[steps:] == episode[-1], kept, torch.zeros((), dtype=x.dtype, device=x.device))
    return y.to(x.dtype), kept


def _plain_scan(s, case, x, dt, B, C, z, resets):
    """``[T, N, ...]`` -> y, last state."""
    dim, groups = case["dim"], case["groups"]
    delta = dt.float() if s["dt_bias"] is None else dt.float() + s["dt_bias"]
    if case["softplus"]:
        delta = delta.clamp_min(0.0) + torch.log1p(torch.exp(-delta.abs()))
    wide = lambda t: t.float().repeat_interleave(dim // groups, dim=2) if groups > 1 else t.float()  # noqa: E731
    decay = torch.exp(delta.unsqueeze(-1) * s["A"])
    if resets is not None:
        decay = torch.where(resets[..., None, None], 0.0, decay)
    push = (delta * x.float()).unsqueeze(-1) * wide(B)
    h, states = s["state"], []
    for a, b in zip(decay.unbind(0), push.unbind(0)):  # the recurrence, step by step
        h = torch.addcmul(b, a, h)
        states.append(h)
    del decay, push
    y = (torch.stack(states) * wide(C)).sum(-1)
    if s["D"] is not None:
        y = y + s["D"] * x.float()
    if z is not None:
        y = y * (z.float() * torch.sigmoid(z.float()))
    return y.to(x.dtype), h


def _plain_noise(index, key):
    """32 bits of an index: two rounds of multiply and shift."""
    h = ((index ^ key) * 0x9E3779B9) & 0xFFFFFFFF
    h = h ^ (h >> 16)
    h = (h * 0x6A09E667) & 0xFFFFFFFF
    return h ^ (h >> 15)


def _plain_round_8(t, noise16, mantissa, least, kind):
    """``t`` to 8 bits, up or down with the odds of its distance: ``noise16``
    are 16 random bits, ``least`` the smallest normal value."""
    cut = 23 - mantissa
    bits = t.abs().view(torch.int32)
    normal = ((bits + (noise16 << (cut - 16))) & ~((1 << cut) - 1)).view(torch.float32)
    quantum = least / (1 << mantissa)
    steps = t.abs() * (1.0 / quantum)
    whole = torch.floor(steps)
    small = (whole + torch.floor((steps - whole) + noise16.float() * 2.0**-16)) * quantum
    return torch.copysign(torch.where(t.abs() < least, small, normal), t).to(kind)


def _plain_adamw(s, case):
    s["step"] += 1
    step, (b1, b2) = s["step"], BETAS
    p, g = s["params"].float(), s["grads"].float()
    m, v = s["exp_avg"], s["exp_avg_sq"]
    small = case["bits"] == 8
    if small:
        m = (m.float().view(-1, STATE_BLOCK) * s["exp_avg_scale"].view(-1, 1)).view(-1)
        v = (v.float().view(-1, STATE_BLOCK) * s["exp_avg_sq_scale"].view(-1, 1)).view(-1)
    m = m * b1 + g * (1 - b1)
    v = v * b2 + g * g * (1 - b2)
    update = (m * (LR / (1 - b1**step))) / (torch.sqrt(v) * (1.0 / math.sqrt(1 - b2**step)) + EPS)
    s["params"].copy_(p * (1 - LR * DECAY) - update)
    if not small:
        s["exp_avg"].copy_(m)
        s["exp_avg_sq"].copy_(v)
        return [s["params"], s["exp_avg"], s["exp_avg_sq"]]
    key = (ADAM_SEED + step * 0x9E3779B9) & 0xFFFFFFFF
    noise = _plain_noise(torch.arange(p.numel(), dtype=torch.int64, device=p.device), key)
    for k, t, top, part, fmt in (
        ("exp_avg", m, E4M3_MAX, noise & 0xFFFF, (3, 2.0**-6, torch.float8_e4m3fn)),
        ("exp_avg_sq", v, E5M2_MAX, noise >> 16, (2, 2.0**-14, torch.float8_e5m2)),
    ):
        t = t.view(-1, STATE_BLOCK)
        most = t.abs().amax(1, keepdim=True).clamp_min(SCALE_FLOOR)
        scaled = (t * (top / most)).clamp(-top, top).view(-1)
        q = _plain_round_8(scaled, part.to(torch.int32), *fmt)
        if k == "exp_avg_sq":  # what is not zero stays so
            q = torch.where(scaled > 0, q.float().clamp_min(2.0**-16), 0.0).to(q.dtype)
        s[k].copy_(q)
        s[k + "_scale"].copy_((most / top).view(-1))
    return [s["params"], s["exp_avg"], s["exp_avg_sq"], s["exp_avg_scale"], s["exp_avg_sq_scale"]]


# ----------------------------------------------------------------- one pass


def _grads(s, outputs, d_outputs):
    leaves = [s[k] for k in LEAVES[s["case"]["kind"]] if s[k] is not None]
    return list(torch.autograd.grad(outputs, leaves, d_outputs))


def _run_norm(s):
    case = s["case"]
    kind, group = case["kind"], case["group"]
    x, weight, residual = s["x"], s["weight"], s["residual"]
    if own:
        from gbxcule_amd.rl import rms_norm, rms_norm_fp8

        if kind == "norm_fp8":
            return list(rms_norm_fp8(x, weight, residual, eps=NORM_EPS, group=group or None))
        out = rms_norm(x, weight, residual, eps=NORM_EPS)
        out = [out] if residual is None else list(out)
    else:
        y, total = _plain_rms_norm(x, weight, residual)
        out = list(_plain_fp8(y, group)) if kind == "norm_fp8" else [y.to(x.dtype)]
        out += [] if residual is None else [total.to(x.dtype)]
    if kind == "norm_train":
        out += _grads(s, out, [s["dy"]] if residual is None else [s["dy"], s["dsummed"]])
    return out


def _run_conv(s):
    case = s["case"]
    args = s["x"], s["weight"], s["bias"]
    if own:
        from gbxcule_amd.rl import causal_conv, causal_conv_step

        options = {"resets": s["resets"], "activation": "silu" if case["silu"] else None}
        if case["kind"] == "conv_step":
            return [causal_conv_step(*args, s["state"], **options), s["state"]]
        y, state = causal_conv(*args, state=s["state"], **options)
    elif case["kind"] == "conv_step":
        resets = None if s["resets"] is None else s["resets"].unsqueeze(0)
        y, state = _plain_conv(s["x"].unsqueeze(0), *args[1:], s["state"].transpose(0, 1), resets, case["silu"])
        s["state"].copy_(state.transpose(0, 1))
        return [y[0], s["state"]]
    else:
        y, state = _plain_conv(*args, s["state"].transpose(0, 1), s["resets"], case["silu"])
        state = state.transpose(0, 1).contiguous()
    out = [y, state]
    if case["kind"] == "conv_train":
        out += _grads(s, [y], [s["dy"]])
    return out


def _run_scan(s):
    case = s["case"]
    if own:
        from gbxcule_amd.rl import selective_scan, selective_scan_step

        args = [s[k] for k in ("x", "dt", "A", "B", "C", "D", "z")]
        options = {"dt_bias": s["dt_bias"], "softplus": case["softplus"], "resets": s["resets"]}
        if case["kind"] == "scan_step":
            return [selective_scan_step(*args, state=s["state"], **options), s["state"]]
        y, state = selective_scan(*args, state=s["state"], **options)
    elif case["kind"] == "scan_step":
        row = {k: None if s[k] is None else s[k].unsqueeze(0) for k in ("x", "dt", "B", "C", "z", "resets")}
        y, state = _plain_scan(s, case, **row)
        s["state"].copy_(state)
        return [y[0], s["state"]]
    else:
        y, state = _plain_scan(s, case, *(s[k] for k in ("x", "dt", "B", "C", "z", "resets")))
    out = [y.detach(), state.detach()]
    if case["kind"] == "scan_train":
        out += _grads(s, [y], [s["dy"]])
    return out


def _run_adamw(s):
    if not own:
        return _plain_adamw(s, s["case"])
    s["opt"].step()
    flat = s["opt"].flat_state()
    return [s["params"], *(flat[k] for k in ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale") if k in flat)]


def run(s):
    kind = s["case"]["kind"].split("_")[0]
    if s["case"]["kind"] in LEAVES:
        return {"norm": _run_norm, "conv": _run_conv, "scan": _run_scan}[kind](s)
    with torch.no_grad():
        return {"norm": _run_norm, "conv": _run_conv, "scan": _run_scan, "adamw": _run_adamw}[kind](s)


# --------------------------------------------------------------------- work


def work(case):
    """Bytes: every input read once and every output written once.
    Operations: a multiplication, an addition or a function each one."""
    kind = case["kind"]
    e = BYTES[case["dtype"]]
    if kind.startswith("norm"):
        n, dim = case["rows"] * case["dim"], case["dim"]
        each = 2 * e if case["residual"] else e  # x and the residual, or x alone
        b = n * each + 4 * dim
        if kind == "norm_fp8":
            b += n * (1 + (e if case["residual"] else 0)) + 4 * case["rows"] * (-(-dim // case["group"]) if case["group"] else 1)
            return {"bytes": b, "flops": 8 * n}
        b += n * each  # y and the sum
        if kind == "norm_train":  # their gradients in; x's and the residual's, which are one, out
            b += n * each + n * e + 4 * dim
        return {"bytes": b, "flops": (16 if kind == "norm_train" else 5) * n}
    if kind.startswith("conv"):
        rows, dim, width = case["steps"] * case["envs"], case["dim"], case["width"]
        b = rows * dim * e * (4 if kind == "conv_train" else 2) + 2 * case["envs"] * (width - 1) * dim * e
        b += dim * (width + 1) * 4 * (2 if kind == "conv_train" else 1) + (rows if case["resets"] else 0)
        return {"bytes": b, "flops": rows * dim * (2 * width + 4) * (3 if kind == "conv_train" else 1)}
    if kind.startswith("scan"):
        rows, dim, states, gs = case["steps"] * case["envs"], case["dim"], case["states"], case["groups"] * case["states"]
        tensors = 4 if case["gate"] else 3  # x, dt, y and the gate
        b = rows * e * (tensors * dim + 2 * gs) + (rows if case["resets"] else 0)
        b += 2 * case["envs"] * dim * states * 4 + dim * (states + 2) * 4
        if kind == "scan_train":  # dy in, the gradients of x, dt, the gate, B and C out
            b += rows * e * (tensors * dim + 2 * gs) + dim * (states + 2) * 4
        return {"bytes": b, "flops": rows * dim * states * (28 if kind == "scan_train" else 7)}
    n = sum(math.prod(sh) for sh in _adamw_shapes(case))
    states = 2 * 2 if case["bits"] == 8 else 2 * 8
    return {"bytes": n * (3 * e + states), "flops": n * (40 if case["bits"] == 8 else 16)}


# ------------------------------------------------------------ 64-bit values


def _exact_norm(case, s):
    x, w = s["x"].double(), s["weight"].double()
    if s["residual"] is not None:  # what is normalised is the sum as the stream carries it
        x = (x + s["residual"].double()).to(s["x"].dtype).double()
    inv = 1.0 / torch.sqrt(torch.mean(x**2, dim=-1, keepdim=True) + NORM_EPS)
    y = w * (x * inv)
    kept = [] if s["residual"] is None else [x]
    if case["kind"] == "norm_fp8":
        size = case["group"] or case["dim"]
        most = torch.stack([part.abs().max(dim=-1).values for part in y.split(size, dim=-1)], dim=-1)
        scale = most / E4M3_MAX
        return [None, scale if case["group"] else scale[:, 0], *kept]
    if case["kind"] == "norm":
        return [y, *kept]
    dy = s["dy"].double()
    dw = torch.sum(dy * x * inv, dim=0)
    gy = w * dy
    dx = inv * gy - x * inv**3 * torch.mean(gy * x, dim=-1, keepdim=True)
    if s["residual"] is None:
        return [y, dx, dw]
    dx = dx + s["dsummed"].double()
    return [y, x, dx, dx, dw]


def _exact_conv(case, s):
    one = case["kind"] == "conv_step"
    x = (s["x"][None] if one else s["x"]).double()
    steps, envs, dim, width = x.shape[0], case["envs"], case["dim"], case["width"]
    resets = s["resets"]
    if resets is not None and one:
        resets = resets[None]
    w, b = s["weight"].double(), 0.0 if s["bias"] is None else s["bias"].double()
    window = list(s["state"].double().unbind(1))  # the inputs before this one, oldest first
    valid = [torch.ones(envs, 1, dtype=torch.float64, device=x.device) for _ in window]
    train = case["kind"] == "conv_train"
    y = torch.empty_like(x)
    dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), torch.zeros(dim, dtype=torch.float64, device=x.device)
    for t in range(steps):
        if resets is not None:
            go = 1.0 - resets[t].double()[:, None]
            valid = [k * go for k in valid]
        taps = [k * u for k, u in zip(valid, window)] + [x[t]]
        pre = b + sum(w[:, i] * u for i, u in enumerate(taps))
        sig = 1.0 / (1.0 + torch.exp(-pre))
        y[t] = pre * sig if case["silu"] else pre
        if train:
            d = s["dy"][t].double()
            if case["silu"]:
                d = d * (sig + pre * sig * (1.0 - sig))
            db += d.sum(0)
            for i, u in enumerate(taps):
                dw[:, i] += (d * u).sum(0)
                back = t - (width - 1 - i)
                if back >= 0:
                    dx[back] += d * w[:, i] * (valid[i] if i < width - 1 else 1.0)
        window, valid = window[1:] + [x[t]], valid[1:] + [torch.ones_like(valid[0])]
    state = torch.stack([k * u for k, u in zip(valid, window)], dim=1)
    out = [y[0] if one else y, state]
    return out + [dx, dw] + ([] if s["bias"] is None else [db]) if train else out


def _exact_scan(case, s):
    one = case["kind"] == "scan_step"
    get = lambda k: None if s[k] is None else (s[k][None] if one else s[k])  # noqa: E731
    x, dt, z, B, C, resets = (get(k) for k in ("x", "dt", "z", "B", "C", "resets"))
    steps, dim, groups = x.shape[0], case["dim"], case["groups"]
    train = case["kind"] == "scan_train"
    A, h = s["A"].double(), s["state"].double()
    bias = 0.0 if s["dt_bias"] is None else s["dt_bias"].double()
    skip = None if s["D"] is None else s["D"].double()

    def at(t):
        raw = dt[t].double() + bias
        delta = torch.where(raw > 40, raw, torch.log1p(torch.exp(raw.clamp_max(40)))) if case["softplus"] else raw
        a = torch.exp(delta[..., None] * A)
        if resets is not None:
            a = a * (1.0 - resets[t].double()[:, None, None])
        spread = lambda v: v[t].double().repeat_interleave(dim // groups, dim=1)  # noqa: E731
        return raw, delta, a, spread(B), spread(C), x[t].double()

    y = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    before = []
    for t in range(steps):
        _, delta, a, b, c, u = at(t)
        if train:
            before.append(h)
        h = a * h + (delta * u)[..., None] * b
        out = (h * c).sum(-1)
        if skip is not None:
            out = out + skip * u
        if z is not None:
            gate = z[t].double()
            out = out * gate / (1.0 + torch.exp(-gate))
        y[t] = out
    if not train:
        return [y[0] if one else y, h]
    last = h
    dx, ddt, dz = torch.empty_like(y), torch.empty_like(y), torch.empty_like(y)
    dA, dD, dbias = torch.zeros_like(A), torch.zeros_like(A[:, 0]), torch.zeros_like(A[:, 0])
    dB = torch.empty(B.shape, dtype=torch.float64, device=x.device)
    dC = torch.empty_like(dB)
    carry = torch.zeros_like(h)  # what the steps after this one ask of the state
    for t in range(steps - 1, -1, -1):
        raw, delta, a, b, c, u = at(t)
        h = a * before[t] + (delta * u)[..., None] * b
        d = s["dy"][t].double()
        if z is not None:
            gate = z[t].double()
            sig = 1.0 / (1.0 + torch.exp(-gate))
            ungated = (h * c).sum(-1) + (0.0 if skip is None else skip * u)
            dz[t] = d * ungated * sig * (1.0 + gate * (1.0 - sig))
            d = d * gate * sig
        shared = lambda v: v.unflatten(1, (groups, -1)).sum(2)  # noqa: E731
        dC[t] = shared(d[..., None] * h)
        carry = carry + d[..., None] * c
        dB[t] = shared(carry * (delta * u)[..., None])
        through = (carry * b).sum(-1)
        by_decay = carry * a * before[t]
        dA += (by_decay * delta[..., None]).sum(0)
        ddelta = through * u + (by_decay * A).sum(-1)
        dx[t] = through * delta + (0.0 if skip is None else skip * d)
        if skip is not None:
            dD += (d * u).sum(0)
        ddt[t] = ddelta / (1.0 + torch.exp(-raw)) if case["softplus"] else ddelta
        dbias += ddt[t].sum(0)
        carry = carry * a
        before[t] = None
    grads = {"x": dx, "dt": ddt, "A": dA, "B": dB, "C": dC, "D": dD, "z": dz, "dt_bias": dbias}
    return [y, last, *(grads[k] for k in LEAVES["scan_train"] if s[k] is not None)]


def _exact_adamw(case, s):
    b1, b2 = BETAS
    step = 10
    p, g = s["params"].double(), s["grads"].double()
    scaled = lambda k: (s[k].float().double().view(-1, STATE_BLOCK) * s[k + "_scale"].double()[:, None]).view(-1)  # noqa: E731
    m, v = (scaled(k) if case["bits"] == 8 else s[k].double() for k in ("exp_avg", "exp_avg_sq"))
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g**2
    p = p - LR * DECAY * p - LR * (m / (1 - b1**step)) / (torch.sqrt(v / (1 - b2**step)) + EPS)
    if case["bits"] == 32:
        return [p, m, v]
    tops = [t.abs().view(-1, STATE_BLOCK).max(1).values.clamp_min(SCALE_FLOOR) for t in (m, v)]
    return [p, None, None, tops[0] / E4M3_MAX, tops[1] / E5M2_MAX]


def exact(case, seed):
    s = _inputs(case, seed)
    with torch.no_grad():
        kind = case["kind"].split("_")[0]
        return {"norm": _exact_norm, "conv": _exact_conv, "scan": _exact_scan, "adamw": _exact_adamw}[kind](case, s)
