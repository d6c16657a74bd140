"""More operators of a policy that remembers, as timed cases.

Beside the selective scan (``perf/operators.py``) a policy's block can carry a
matrix for each head that it corrects at every step: the gated delta rule
(``delta_rule``).  ``layer_norm`` opens such a block and ``sample_actions``
turns the policy's logits into actions.  Everything is time-major as in
``RolloutBuffer``: ``[steps, envs, heads, channels]``, and ``resets[t, n]`` says
that env ``n`` begins an episode at step ``t``.

The actor makes one step of all envs at a time, from a handful of envs to
thousands; the learner reads whole rollouts forward and backward; an evaluation
runs one long recorded episode as a prompt.

With ``own`` false, ``run`` computes the operators with elementary torch
operations in 32 bits (sampling in 64: a random number may fall next to a
border between two actions), rounded once at the end.  With ``own`` true it
calls the framework.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
NORM_EPS = 1e-5
UNIT_EPS = 1e-6  # added to a squared length before its root
STILL = 0.25  # of the steps show what the step before showed


def _norm(name, kind, rows, dim, dtype="bf16", residual=True, bias=True):
    return {"name": name, "kind": kind, "rows": rows, "dim": dim, "dtype": dtype, "residual": residual, "bias": bias}


def _delta(name, kind, steps, envs, heads, keys=64, values=64, share=1, dtype="bf16", resets=0.0, normalize=True):
    return {"name": name, "kind": kind, "steps": steps, "envs": envs, "heads": heads, "keys": keys, "values": values,
            "share": share, "dtype": dtype, "resets": resets, "normalize": normalize}  # fmt: skip


def _sample(name, rows, actions, dtype="f32", temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, per_row=False, masked=0.0):
    return {"name": name, "kind": "sample", "rows": rows, "actions": actions, "dtype": dtype, "temperature": temperature,
            "top_k": top_k, "top_p": top_p, "min_p": min_p, "per_row": per_row, "masked": masked}  # fmt: skip


def listed():
    return [
        # acting with 64 envs: one row an env, launch latency
        _norm("layer_norm_act_64", "norm", 64, 256),
        # a learner's minibatch of 128 steps x 1,024 envs, forward and backward
        _norm("layer_norm_train_131072", "norm_train", 131_072, 512),
        # the same at a ragged env count and an odd width, in 32 bits, the block's first norm
        _norm("layer_norm_train_20011", "norm_train", 20_011, 1023, dtype="f32", residual=False),
        # one step of a handful of envs
        _delta("delta_step_64", "delta_step", 1, 64, 4, resets=0.01),
        # one step of 8,192 envs: half a gigabyte of state read and written
        _delta("delta_step_8192", "delta_step", 1, 8192, 4, resets=0.01),
        # one recorded episode of 8,192 steps as a prompt: one row, a long axis
        _delta("delta_prompt_8192", "delta", 8192, 1, 8),
        # the learner's recurrence over a rollout, forward and backward
        _delta("delta_train_128x1024", "delta_train", 128, 1024, 4, resets=0.01),
        # wide heads, two of values for each of keys
        _delta("delta_train_64x256_wide", "delta_train", 64, 256, 4, keys=128, values=128, share=2, resets=0.01),
        # odd sizes in 32 bits
        _delta("delta_train_77x37", "delta_train", 77, 37, 3, keys=40, values=56, dtype="f32", resets=0.05),
        # an action for each of 64 envs from the policy's own distribution
        _sample("sample_act_64x8", 64, 8),
        # an action for each of 131,072 envs, each with its own temperature and cuts, some buttons not allowed
        _sample("sample_131072x8", 131_072, 8, per_row=True, masked=0.1),
        # sequences of inputs as actions: a long row, cut to the likely ones
        _sample("sample_512x32768", 512, 32_768, dtype="bf16", temperature=0.8, top_k=50, top_p=0.95, min_p=0.01),
    ]  # fmt: skip


def _log_int(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def _channels(rng, lo, hi):
    """A channel count: mostly one that 16-byte loads take, else any."""
    d = _log_int(rng, lo, hi)
    return max(8, d - d % 8) if rng.random() < 0.6 else d


def draw(rng):
    kind = rng.choice(["norm", "norm_train", "delta", "delta_train", "delta_train", "delta_step", "sample", "sample"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind.startswith("norm"):
        dim = _channels(rng, 24, 8192)
        rows = _log_int(rng, 1, min(131_072, 131_072 * 512 // dim))
        return _drawn(_norm("", kind, rows, dim, dtype, rng.random() < 0.7, rng.random() < 0.7))
    if kind.startswith("delta"):
        resets = rng.choice([0.0, 0.005, 0.01, 0.05])
        share = rng.choice([1, 1, 2, 4])
        heads = share * rng.choice([1, 2, 3, 4])
        keys, values = _channels(rng, 16, 128), _channels(rng, 16, 128)
        size = heads * keys * values
        if kind == "delta_step":
            steps, envs = 1, _log_int(rng, 1, max(1, 8192 * 4 * 64 * 64 // size))
        elif kind == "delta":
            steps = _log_int(rng, 1, 8192)
            envs = _log_int(rng, 1, max(1, min(4096, 128 * 1024 * 4 * 64 * 64 // (4 * steps * size))))
        else:
            steps = _log_int(rng, 1, 512)
            envs = _log_int(rng, 1, max(1, min(4096, 128 * 1024 * 4 * 64 * 64 // (2 * steps * size))))
        return _drawn(_delta("", kind, steps, envs, heads, keys, values, share, dtype, resets, rng.random() < 0.8))
    actions = _log_int(rng, 2, 32_768)
    rows = _log_int(rng, 1, min(131_072, 512 * 32_768 // actions))
    return _drawn(
        _sample("", rows, actions, rng.choice(["f32", "bf16", "f16"]), rng.choice([0.0, 0.5, 0.8, 1.0, 1.3]),
                rng.choice([0, 0, 1, 5, 40, 200]), rng.choice([1.0, 0.99, 0.9, 0.5]), rng.choice([0.0, 0.0, 0.02, 0.1]),
                rng.random() < 0.4, rng.choice([0.0, 0.2])))  # fmt: skip


def _drawn(case):
    return {k: v for k, v in case.items() if k != "name"}


# ------------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 13)


def _randn(gen, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, device="cuda", generator=gen) * scale).to(dtype)


def _rand(gen, *shape):
    return torch.rand(shape, device="cuda", generator=gen)


def _norm_inputs(case, seed):
    gen, dtype = _gen(seed), DTYPES[case["dtype"]]
    shape = (case["rows"], case["dim"])
    s = {"x": _randn(gen, *shape, dtype=dtype), "weight": 1.0 + _randn(gen, case["dim"], scale=0.1)}
    s["bias"] = _randn(gen, case["dim"], scale=0.1) if case["bias"] else None
    # a residual stream has grown over the blocks before, and its channels have means of their own
    s["residual"] = (_randn(gen, *shape, scale=3.0) + _randn(gen, case["dim"])).to(dtype) if case["residual"] else None
    if case["kind"] == "norm_train":
        s["dy"] = _randn(gen, *shape, dtype=dtype)
        s["dsummed"] = _randn(gen, *shape, dtype=dtype) if case["residual"] else None
    return s


def _delta_inputs(case, seed):
    gen, dtype = _gen(seed), DTYPES[case["dtype"]]
    steps, envs, heads, keys, values = (case[k] for k in ("steps", "envs", "heads", "keys", "values"))
    shared = heads // case["share"]
    # q, k and v are parts of one projection's output; the screen stands still now and then, and so do they
    wide = torch.randn(steps, envs, 2 * shared * keys + heads * values, device="cuda", generator=gen)
    if not case["normalize"]:
        wide[..., : 2 * shared * keys] *= keys**-0.5
    moved = torch.where(_rand(gen, steps, envs) < STILL, 0, torch.arange(steps, device="cuda")[:, None])
    moved = moved.cummax(0).values
    wide = wide.to(dtype)[moved, torch.arange(envs, device="cuda")]
    q, k, v = wide.split([shared * keys, shared * keys, heads * values], dim=-1)
    s = {"q": q.unflatten(-1, (shared, keys)), "k": k.unflatten(-1, (shared, keys)), "v": v.unflatten(-1, (heads, values))}
    # rates of 1 to 16 times step sizes of 0.001 to 0.1, as the layer computes them in 32 bits
    rate = 1.0 + 15.0 * _rand(gen, heads)
    size = 0.001 * 100.0 ** _rand(gen, heads)
    s["g"] = -rate * size * torch.exp(_randn(gen, steps, envs, heads, scale=0.5))
    s["beta"] = torch.sigmoid(_randn(gen, steps, envs, heads, scale=1.5))
    s["state"] = _randn(gen, envs, heads, keys, values, scale=0.3)
    s["resets"] = _rand(gen, steps, envs) < case["resets"] if case["resets"] > 0 else None
    if case["kind"] == "delta_train":
        s["dy"] = _randn(gen, steps, envs, heads, values, dtype=dtype)
    if case["kind"] == "delta_step":
        for name in ("q", "k", "v", "g", "beta", "resets"):
            s[name] = None if s[name] is None else s[name][0]
    return s


def _sample_inputs(case, seed):
    gen, dtype = _gen(seed), DTYPES[case["dtype"]]
    rows, actions = case["rows"], case["actions"]
    # some envs are sure of what to do, others are not
    logits = _randn(gen, rows, actions) * (0.3 * 20.0 ** _rand(gen, rows, 1))
    if case["masked"] > 0:  # the last action is always allowed
        barred = _rand(gen, rows, actions) < case["masked"]
        barred[:, -1] = False
        logits = logits.masked_fill(barred, -math.inf)
    s = {"logits": logits.to(dtype), "uniform": _rand(gen, rows)}
    for name in ("temperature", "top_k", "top_p", "min_p"):
        s[name] = case[name]
    if case["per_row"]:  # a ladder of explorers, greedy ones among them
        pick = lambda values, kind: torch.tensor(values, dtype=kind, device="cuda")[  # noqa: E731
            torch.randint(len(values), (rows,), device="cuda", generator=gen)]  # fmt: skip
        s["temperature"] = pick([0.0, 0.5, 0.9, 1.0, 1.5], torch.float32)
        s["top_k"] = pick([0, 1, 3, 6, 50], torch.int32)
        s["top_p"] = pick([1.0, 0.95, 0.8, 0.3], torch.float32)
        s["min_p"] = pick([0.0, 0.05, 0.2], torch.float32)
    return s


INPUTS = {"norm": _norm_inputs, "delta": _delta_inputs, "sample": _sample_inputs}

#: What a training step differentiates.
LEAVES = {
    "norm_train": ("x", "residual", "weight", "bias"),
    "delta_train": ("q", "k", "v", "g", "beta"),
}


def _family(case):
    return case["kind"].split("_")[0]


def prepare(case, seed):
    s = INPUTS[_family(case)](case, seed)
    s["case"] = case
    for k in LEAVES.get(case["kind"], ()):
        s[k] = None if s[k] is None else s[k].detach().requires_grad_()
    return s


# --------------------------------------------------------------- plain forms


def _plain_layer_norm(x, weight, bias, residual):
    total = x.float() if residual is None else (x.float() + residual.float()).to(x.dtype).float()
    centred = total - total.mean(-1, keepdim=True)
    y = centred * torch.rsqrt((centred * centred).mean(-1, keepdim=True) + NORM_EPS) * weight
    return y if bias is None else y + bias, total


def _plain_unit(t, normalize):
    t = t.float()
    return t * torch.rsqrt((t * t).sum(-1, keepdim=True) + UNIT_EPS) if normalize else t


def _plain_delta(case, q, k, v, g, beta, state, resets):
    """``[T, N, ...]`` -> y, last state."""
    share = case["share"]
    q, k = (_plain_unit(t, case["normalize"]).repeat_interleave(share, dim=2) for t in (q, k))
    q = (q * case["keys"] ** -0.5).unsqueeze(-1)
    k, v, beta = k.unsqueeze(-1), v.float().unsqueeze(-2), beta[..., None, None]
    decay = torch.exp(g)
    if resets is not None:
        decay = torch.where(resets[..., None], 0.0, decay)
    decay, out = decay[..., None, None], []
    for t in range(len(q)):  # the recurrence, step by step
        state = state * decay[t]
        error = (v[t] - (state * k[t]).sum(-2, keepdim=True)) * beta[t]
        state = torch.addcmul(state, k[t], error)
        out.append((state * q[t]).sum(-2))
    return torch.stack(out), state


def _column(value, rows, device):
    """An option as a column with one value a row, in 64 bits."""
    if isinstance(value, torch.Tensor):
        return value.double().unsqueeze(-1)
    return torch.full((rows, 1), float(value), dtype=torch.float64, device=device)


def _plain_sample(s):
    logits, n = s["logits"].double(), s["logits"].shape[1]
    heat, top_k, top_p, min_p = (_column(s[k], len(logits), logits.device) for k in ("temperature", "top_k", "top_p", "min_p"))
    shifted = logits - logits.amax(-1, keepdim=True)
    weight = torch.where(heat > 0, torch.exp(shifted / torch.where(heat > 0, heat, 1.0)), (shifted == 0).double())
    # likeliest first, the lowest of equals before the others
    order = torch.sort(logits, dim=-1, descending=True, stable=True).indices
    ranked = weight.gather(-1, order)
    place = torch.arange(n, device=logits.device)
    top_k = torch.where(heat > 0, torch.where(top_k > 0, top_k, n), 1)
    ranked = torch.where(place < top_k, ranked, 0.0)
    running = ranked.cumsum(-1)
    before = running - ranked
    kept = (place < top_k) & ((top_p >= 1.0) | (before < top_p * running[:, -1:])) & (ranked >= min_p)
    kept[:, 0] = True
    weight = torch.zeros_like(weight).scatter(-1, order, torch.where(kept, ranked, 0.0))
    running = weight.cumsum(-1)
    total = running[:, -1:]
    past = (running > s["uniform"].double().unsqueeze(-1) * total) & (weight > 0)
    action = torch.where(past.any(-1), past.int().argmax(-1), n - 1)
    logp = torch.log(weight.gather(-1, action.unsqueeze(-1)) / total).squeeze(-1)
    return action.to(torch.int32), logp.float()


# ----------------------------------------------------------------- one pass


def _grads(s, outputs, d_outputs):
    leaves = [s[k] for k in LEAVES[s["case"]["kind"]] if s[k] is not None]
    return list(torch.autograd.grad(outputs, leaves, d_outputs))


def _run_norm(s):
    x, residual = s["x"], s["residual"]
    if own:
        from gbxcule_amd.rl import layer_norm

        out = layer_norm(x, s["weight"], s["bias"], residual, eps=NORM_EPS)
        out = [out] if residual is None else list(out)
    else:
        y, total = _plain_layer_norm(x, s["weight"], s["bias"], residual)
        out = [y.to(x.dtype)] + ([] if residual is None else [total.to(x.dtype)])
    if s["case"]["kind"] == "norm_train":
        out = [t.detach() for t in out] + _grads(s, out, [s["dy"]] if residual is None else [s["dy"], s["dsummed"]])
    return out


def _run_delta(s):
    case = s["case"]
    rows = [s[k] for k in ("q", "k", "v", "g", "beta")]
    if own:
        from gbxcule_amd.rl import delta_rule, delta_rule_step

        options = {"normalize": case["normalize"], "resets": s["resets"]}
        if case["kind"] == "delta_step":
            return [delta_rule_step(*rows, state=s["state"], **options), s["state"]]
        y, state = delta_rule(*rows, state=s["state"], **options)
    elif case["kind"] == "delta_step":
        y, state = _plain_delta(case, *(t.unsqueeze(0) for t in rows), s["state"], None if s["resets"] is None else s["resets"].unsqueeze(0))
        s["state"].copy_(state)
        return [y[0].to(rows[2].dtype), s["state"]]
    else:
        y, state = _plain_delta(case, *rows, s["state"], s["resets"])
        y = y.to(rows[2].dtype)
    out = [y.detach(), state.detach()]
    if case["kind"] == "delta_train":
        out += _grads(s, [y], [s["dy"]])
    return out


def _run_sample(s):
    if not own:
        return list(_plain_sample(s))
    from gbxcule_amd.rl import sample_actions

    return list(sample_actions(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"]))


RUN = {"norm": _run_norm, "delta": _run_delta, "sample": _run_sample}


def run(s):
    one = RUN[_family(s["case"])]
    if s["case"]["kind"] in LEAVES:
        return one(s)
    with torch.no_grad():
        return one(s)


# --------------------------------------------------------------------- work


def work(case):
    """Bytes: every input read once and every output written once.
    Operations: a multiplication, an addition or a function each one; the
    delta rule's as its formulas have them, step by step."""
    kind = case["kind"]
    e = BYTES[case["dtype"]]
    if kind.startswith("norm"):
        n, dim, train = case["rows"] * case["dim"], case["dim"], kind == "norm_train"
        each = 2 * e if case["residual"] else e  # x and the residual, or x alone
        params = 4 * dim * (2 if case["bias"] else 1)
        b = 2 * n * each + params  # y and the sum out
        if train:  # their gradients in; x's and the residual's, which are one, out
            b += n * each + n * e + params
        return {"bytes": b, "flops": (22 if train else 8) * n}
    if kind == "sample":
        options = 16 * case["rows"] if case["per_row"] else 0
        return {"bytes": case["rows"] * (case["actions"] * e + 12) + options, "flops": 4 * case["rows"] * case["actions"]}
    rows, heads, keys, values = case["steps"] * case["envs"], case["heads"], case["keys"], case["values"]
    shared = heads // case["share"]
    inputs = rows * (e * (2 * shared * keys + heads * values) + 8 * heads)
    b = inputs + rows * heads * values * e + 8 * case["envs"] * heads * keys * values + (rows if case["resets"] else 0)
    if kind == "delta_train":
        b += inputs + rows * heads * values * e  # dy in, five gradients out
    return {"bytes": b, "flops": rows * heads * keys * values * (21 if kind == "delta_train" else 7)}


# ------------------------------------------------------------ 64-bit values


def _exact_norm(case, s):
    x, w = s["x"].double(), s["weight"].double()
    if s["residual"] is not None:  # what is normalised is the sum as the stream carries it
        x = (x + s["residual"].double()).to(s["x"].dtype).double()
    mean = torch.mean(x, dim=-1, keepdim=True)
    inv = 1.0 / torch.sqrt(torch.mean(x**2, dim=-1, keepdim=True) - mean**2 + NORM_EPS)
    hat = (x - mean) * inv
    y = w * hat + (0.0 if s["bias"] is None else s["bias"].double())
    kept = [] if s["residual"] is None else [x]
    if case["kind"] == "norm":
        return [y, *kept]
    dy = s["dy"].double()
    gy = w * dy
    dx = inv * (gy - torch.mean(gy, dim=-1, keepdim=True) - hat * torch.mean(gy * hat, dim=-1, keepdim=True))
    if s["residual"] is not None:
        dx = dx + s["dsummed"].double()
    grads = [dx] if s["residual"] is None else [dx, dx]
    grads.append(torch.sum(dy * hat, dim=0))
    if s["bias"] is not None:
        grads.append(torch.sum(dy, dim=0))
    return [y, *kept, *grads]


def _exact_delta(case, s):
    """The state before each step is kept, and the steps are walked back by the
    formulas of the derivative, all as products of matrices."""
    one, train = case["kind"] == "delta_step", case["kind"] == "delta_train"
    get = lambda k: None if s[k] is None else (s[k][None] if one else s[k])  # noqa: E731
    q, k, v, g, beta, resets = (get(name) for name in ("q", "k", "v", "g", "beta", "resets"))
    steps, share, scale = q.shape[0], case["share"], 1.0 / math.sqrt(case["keys"])

    def unit(t):
        t = t.double()
        return t / torch.sqrt(t.pow(2).sum(-1, keepdim=True) + UNIT_EPS) if case["normalize"] else t

    def at(t):
        keep = torch.exp(g[t].double())
        if resets is not None:
            keep = keep.masked_fill(resets[t].bool()[:, None], 0.0)
        spread = lambda u: unit(u[t]).repeat_interleave(share, dim=1)  # noqa: E731
        return spread(q) * scale, spread(k), v[t].double(), keep[..., None, None], beta[t].double()[..., None]

    state, before, y = s["state"].double(), [], []
    for t in range(steps):
        qt, kt, vt, keep, bt = at(t)
        if train:
            before.append(state)
        recalled = (kt.unsqueeze(-2) @ state).squeeze(-2) * keep.squeeze(-1)
        state = keep * state + kt.unsqueeze(-1) @ (bt * (vt - recalled)).unsqueeze(-2)
        y.append((qt.unsqueeze(-2) @ state).squeeze(-2))
    y = torch.stack(y)
    if not train:
        return [y[0] if one else y, state]
    last, wide = state, torch.zeros_like(state)  # what the later steps ask of the state
    dq, dk = (torch.zeros(t.shape, dtype=torch.float64, device=y.device) for t in (q, k))
    dv, dg, db = (torch.zeros(t.shape, dtype=torch.float64, device=y.device) for t in (v, g, beta))

    def shared(d, t):  # back through the heads that share a row and its length
        d = d.unflatten(1, (-1, share)).sum(2)
        if not case["normalize"]:
            return d
        t = t.double()
        size = torch.sqrt(t.pow(2).sum(-1, keepdim=True) + UNIT_EPS)
        return d / size - t * (d * t).sum(-1, keepdim=True) / size**3

    for t in range(steps - 1, -1, -1):
        qt, kt, vt, keep, bt = at(t)
        decayed = keep * before[t]
        recalled = (kt.unsqueeze(-2) @ decayed).squeeze(-2)
        error = bt * (vt - recalled)
        after = decayed + kt.unsqueeze(-1) @ error.unsqueeze(-2)
        dy = s["dy"][t].double()
        dq[t] = shared(scale * (after @ dy.unsqueeze(-1)).squeeze(-1), q[t])
        wide = wide + qt.unsqueeze(-1) @ dy.unsqueeze(-2)
        derror = (kt.unsqueeze(-2) @ wide).squeeze(-2)
        dv[t] = bt * derror
        db[t] = (derror * (vt - recalled)).sum(-1)
        dk[t] = shared((wide @ error.unsqueeze(-1)).squeeze(-1) - (decayed @ dv[t].unsqueeze(-1)).squeeze(-1), k[t])
        wide = wide - kt.unsqueeze(-1) @ dv[t].unsqueeze(-2)
        dg[t] = (wide * decayed).sum((-2, -1))
        wide = wide * keep
        before[t] = None
    return [y, last, dq, dk, dv, dg, db]


def _exact_sample(case, s):
    """Cuts as the least value that stays and how many of its equals do; no order of indices."""
    logits = s["logits"].double()
    rows, n = logits.shape
    option = lambda k: s[k].double() if isinstance(s[k], torch.Tensor) else logits.new_full((rows,), float(s[k]))  # noqa: E731
    heat, top_k, top_p, min_p = (option(k) for k in ("temperature", "top_k", "top_p", "min_p"))
    greedy = heat <= 0
    scaled = torch.exp((logits - logits.max(-1, keepdim=True).values) / torch.where(greedy, 1.0, heat)[:, None])
    count = torch.where(greedy, 1.0, torch.where(top_k > 0, top_k.clamp_max(n), float(n)))
    falling = torch.flip(scaled.sort(-1).values, [-1])
    sums = torch.cat([torch.zeros_like(falling[:, :1]), falling.cumsum(-1)], -1)
    mass = sums.gather(-1, count.long()[:, None])
    enough = (sums[:, :-1] < top_p[:, None] * mass).sum(-1).double()
    count = torch.minimum(count, torch.where(top_p >= 1.0, float(n), enough))
    count = torch.minimum(count, (falling >= min_p[:, None]).sum(-1).double()).clamp_min(1.0)
    least = falling.gather(-1, count.long()[:, None] - 1)
    equal = scaled == least
    spare = count[:, None] - (scaled > least).sum(-1, keepdim=True)
    kept = (scaled > least) | (equal & (equal.cumsum(-1) <= spare))
    scaled = torch.where(kept, scaled, 0.0)
    running = scaled.cumsum(-1)
    action = (running <= s["uniform"].double()[:, None] * running[:, -1:]).sum(-1).clamp_max(n - 1)
    logp = scaled.gather(-1, action[:, None]).log() - running[:, -1:].log()
    return [action.to(torch.int32), logp.squeeze(-1)]


def exact(case, seed):
    s = INPUTS[_family(case)](case, seed)
    with torch.no_grad():
        return {"norm": _exact_norm, "delta": _exact_delta, "sample": _exact_sample}[_family(case)](case, s)
