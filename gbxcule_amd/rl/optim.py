"""AdamW over all of a policy's tensors in a few launches.

The moments of a parameter group lie in flat buffers, tensor after tensor,
each from a multiple of 256 elements.  With ``state_bits=8`` the first moment
is ``torch.float8_e4m3fn`` and the second ``torch.float8_e5m2``, each with a
float32 scale for every 256 elements (the largest absolute value maps to the
format's largest), 2 bytes an element and 1/32 more for the scales in place of
8.  They are rounded up or down with the odds of the distance, by a hash of
the element's group and place, the step and ``seed``: rounding to the nearest
would hold a second moment still, since with beta2 = 0.999 a step changes it by
less than half of what 8 bits resolve.  A second moment that is not zero is kept
from rounding to zero.
"""

from __future__ import annotations

import math
from collections import defaultdict

import torch
from torch.optim.optimizer import _global_optimizer_post_hooks, _global_optimizer_pre_hooks

from .._torch_ops import ext

STATE_BLOCK = 256
KINDS = (torch.float32, torch.bfloat16, torch.float16)
# between the rounding keys of two steps, and of two groups' equal places: the
# fractions of the golden ratio and of the square root of 3
_GOLDEN, _ROOT3 = 0x9E3779B9, 0xBB67AE85


class AdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) with one pass over the data.

    Parameters are CUDA tensors of one device, float32, bfloat16 or float16,
    contiguous; gradients of the parameter's type or float32.  The update is
    computed in 32 bits and the parameter rounded once.  ``step`` reads the
    bias corrections on the host, so it is refused under stream capture."""

    def __init__(self, params, lr: float = 1e-3, betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, *, state_bits: int = 32, seed: int = 0) -> None:  # fmt: skip
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
        if not lr >= 0.0 or not eps > 0.0 or not weight_decay >= 0.0:
            raise ValueError(f"lr and weight_decay must not be negative and eps positive, got {lr}, {weight_decay}, {eps}")
        if not all(0.0 <= b < 1.0 for b in betas):
            raise ValueError(f"betas must lie in [0, 1), got {betas}")
        self.state_bits, self.seed = int(state_bits), int(seed)
        self._flat: list[dict[str, torch.Tensor]] = []
        self._plans: list = []  # by parameter group, as self._flat
        self._states: list[list[dict]] = []  # self.state of a group's parameters
        super().__init__(params, {"lr": lr, "betas": tuple(betas), "eps": eps, "weight_decay": weight_decay})

    def add_param_group(self, param_group) -> None:
        super().add_param_group(param_group)
        params = self.param_groups[-1]["params"]
        try:
            self._lay_out(params)
        except Exception:
            self.param_groups.pop()
            raise

    def _lay_out(self, params) -> None:
        device = params[0].device
        for p in params:
            if p.dtype not in KINDS or not p.is_cuda or p.device != device or not p.is_contiguous():
                raise ValueError(f"parameters must be contiguous CUDA tensors of one device in float32, bfloat16 or "
                                 f"float16, got {p.dtype} on {p.device}")  # fmt: skip
        starts, total = [], 0
        for p in params:
            starts.append(total)
            total += -(-p.numel() // STATE_BLOCK) * STATE_BLOCK
        small = self.state_bits == 8
        kinds = (torch.float8_e4m3fn, torch.float8_e5m2) if small else (torch.float32, torch.float32)
        flat = {}
        for key, kind in zip(("exp_avg", "exp_avg_sq"), kinds):
            flat[key] = torch.zeros(total * kind.itemsize, dtype=torch.uint8, device=device).view(kind)
            if small:
                flat[key + "_scale"] = torch.zeros(total // STATE_BLOCK, dtype=torch.float32, device=device)
        self._flat.append(flat)
        keys = ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")
        self._plans.append(ext.AdamwPlan([p.numel() for p in params], starts, *(flat.get(k) for k in keys)))
        self._states.append([self.state[p] for p in params])
        for p, at, state in zip(params, starts, self._states[-1]):
            state["step"] = 0
            for key, t in flat.items():
                if key.endswith("_scale"):
                    state[key] = t[at // STATE_BLOCK : at // STATE_BLOCK - (-p.numel() // STATE_BLOCK)]
                else:
                    state[key] = t[at : at + p.numel()].view(p.shape)

    def flat_state(self, group: int = 0) -> dict[str, torch.Tensor]:
        """A group's moments (and scales) as they lie: every tensor's from the
        next multiple of 256 elements.  Views: they change with ``step``."""
        return dict(self._flat[group])

    def load_flat_state(self, step: int, state: dict[str, torch.Tensor], group: int = 0) -> None:
        """Copies what ``flat_state`` returned, after ``step`` steps."""
        flat = self._flat[group]
        if set(state) != set(flat):
            raise ValueError(f"expected {sorted(flat)}, got {sorted(state)}")
        for key, t in state.items():
            if t.dtype is not flat[key].dtype or t.shape != flat[key].shape:
                raise ValueError(f"{key}: expected {flat[key].dtype} {tuple(flat[key].shape)}, got {t.dtype} {tuple(t.shape)}")
        for key, t in state.items():
            flat[key].copy_(t)
        for p in self.param_groups[group]["params"]:
            self.state[p]["step"] = int(step)

    def __getstate__(self):
        # (pickle takes 8-bit moments as bytes only)
        plain = lambda t: t.view(torch.uint8) if torch.is_tensor(t) and t.itemsize == 1 else t  # noqa: E731
        state = {p: {key: plain(t) for key, t in s.items()} for p, s in self.state.items()}
        return {**super().__getstate__(), "state": state, "state_bits": self.state_bits, "seed": self.seed}

    def __setstate__(self, state) -> None:
        """Copies (``copy.deepcopy``, pickle) get flat buffers of their own."""
        super().__setstate__(state)
        kept, self.state = self.state, defaultdict(dict)
        self._flat, self._plans, self._states = [], [], []
        for group in self.param_groups:
            self._lay_out(group["params"])
            for p, mine in zip(group["params"], self._states[-1]):
                _copy_state(mine, {key: kept[p][key] if key == "step" else kept[p][key].view(t.dtype) for key, t in mine.items()})

    def state_dict(self):
        """As torch's, with ``state_bits`` and ``seed``."""
        return {**super().state_dict(), "state_bits": self.state_bits, "seed": self.seed}

    def load_state_dict(self, state_dict) -> None:
        """Copies the moments into the flat buffers; hyperparameters and the
        hooks on loading as torch does.  A state that does not fit raises
        ``ValueError`` and changes nothing."""
        state_dict = dict(state_dict)
        for hook in self._optimizer_load_state_dict_pre_hooks.values():
            changed = hook(self, state_dict)
            state_dict = state_dict if changed is None else changed
        absent = {"param_groups", "state", "state_bits", "seed"} - set(state_dict)
        if absent:
            raise ValueError(f"the state has no {', '.join(sorted(absent))}")
        groups, saved = self.param_groups, state_dict["param_groups"]
        if state_dict["state_bits"] != self.state_bits:
            raise ValueError(f"a state of {state_dict['state_bits']} bits does not fit state_bits={self.state_bits}")
        if [len(g["params"]) for g in groups] != [len(g["params"]) for g in saved]:
            raise ValueError("the state's parameter groups are not this optimizer's")
        plan = []
        for g, s in zip(groups, saved):
            for p, index in zip(g["params"], s["params"]):
                mine, theirs = self.state[p], state_dict["state"].get(index, {})
                for key, t in mine.items():
                    if key not in theirs:
                        raise ValueError(f"the state has no {key} of parameter {index}")
                    if key != "step" and (theirs[key].shape != t.shape or theirs[key].dtype is not t.dtype):
                        raise ValueError(f"{key} of parameter {index} has another shape or type")
                plan.append((mine, theirs))
        for mine, theirs in plan:
            _copy_state(mine, theirs)
        for g, s in zip(groups, saved):
            g.update({k: v for k, v in s.items() if k != "params"})
        self.seed = int(state_dict["seed"])
        for hook in self._optimizer_load_state_dict_post_hooks.values():
            hook(self)

    def step(self, closure=None, *, grad_scale: torch.Tensor | None = None):
        """One update of every parameter that has a gradient.  ``grad_scale``
        (float32, one element, on the device) multiplies the gradients, such as
        a clipping factor that never leaves the GPU.

        Hooks on the step run, and a profiler sees it, as with torch's own
        optimizers.  Torch's wrapper for both is called only where there are
        any: it takes as long as the rest of a small policy's step on the host."""
        if (self._optimizer_step_pre_hooks or self._optimizer_step_post_hooks or _global_optimizer_pre_hooks
                or _global_optimizer_post_hooks or torch.autograd._profiler_enabled()):  # fmt: skip
            return _hooked_step(self, closure, grad_scale=grad_scale)
        return self._step(closure, grad_scale=grad_scale)

    step.hooked = True  # or torch would wrap it for every call

    def _step(self, closure=None, *, grad_scale: torch.Tensor | None = None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW.step reads its bias corrections on the host: it cannot be captured")
        for g, group in enumerate(self.param_groups):
            self._step_group(g, group, grad_scale)
        return loss

    def _step_group(self, g: int, group, grad_scale) -> None:
        states = self._states[g]
        done = states[0]["step"]
        if all(s["step"] == done for s in states) and self._launch(g, group, grad_scale, (), done + 1):
            for s in states:
                s["step"] = done + 1
            return
        # tensors that a launch can take together: same types, same count of steps
        batches: dict[tuple, list[int]] = {}
        for i, (p, s) in enumerate(zip(group["params"], states)):
            if p.grad is not None:
                batches.setdefault((p.dtype, p.grad.dtype, s["step"]), []).append(i)
        for (_, _, done), which in batches.items():
            if not self._launch(g, group, grad_scale, which, done + 1):
                raise RuntimeError("a gradient changed during the step")
            for i in which:
                states[i]["step"] = done + 1

    def _launch(self, g: int, group, grad_scale, which, step: int) -> bool:
        (b1, b2), lr = group["betas"], float(group["lr"])
        return self._plans[g].step(
            group["params"], which, grad_scale, b1, b2, lr / (1 - b1**step), 1.0 / math.sqrt(1 - b2**step),
            group["eps"], 1 - lr * group["weight_decay"], (self.seed + step * _GOLDEN + g * _ROOT3) & 0xFFFFFFFF,
        )  # fmt: skip


def _copy_state(mine: dict, theirs: dict) -> None:
    """A parameter's step and moments, into the views of the flat buffers."""
    for key, t in mine.items():
        if key != "step":
            t.copy_(theirs[key])
    mine["step"] = int(theirs["step"])


_hooked_step = torch.optim.Optimizer.profile_hook_step(AdamW._step)
