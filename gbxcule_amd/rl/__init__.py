"""RL-side plumbing around the HIP backend: the zero-copy rollout pattern of
the reference's RL engines (``src/gbxcule/rl/``) -- preallocated rollout
buffers, double-buffer stream coordination, packed-pixel helpers and a
game-agnostic packed-pixel env that chains step -> render into a rollout slot
-> RAM senses -> masked reset on torch's current stream with no host sync --
and the operators of a policy that remembers its episode: norms, causal
convolution, selective scan, gated delta rule, the drawing of actions, and the
optimizer that trains it."""

from .async_buffers import AsyncPPOBufferManager, AsyncPPOBufferState
from .env import PackedPixelEnv, collect_rollout
from .packed import (
    get_diff_lut,
    get_unpack_lut,
    pack_2bpp_u8,
    packed_l1_distance,
    unpack_2bpp_u8,
)
from .rollout import RolloutBuffer

# Loaded on first use: these modules import torch and the operators' libraries,
# the others only where they run.  Not in __all__, which a star import would load.
_LAZY = {
    "AdamW": "optim",
    "causal_conv": "ops",
    "causal_conv_step": "ops",
    "delta_rule": "ops",
    "delta_rule_step": "ops",
    "layer_norm": "ops",
    "rms_norm": "ops",
    "rms_norm_fp8": "ops",
    "sample_actions": "ops",
    "selective_scan": "ops",
    "selective_scan_step": "ops",
}

__all__ = [
    "AsyncPPOBufferManager",
    "AsyncPPOBufferState",
    "PackedPixelEnv",
    "RolloutBuffer",
    "collect_rollout",
    "get_diff_lut",
    "get_unpack_lut",
    "pack_2bpp_u8",
    "packed_l1_distance",
    "unpack_2bpp_u8",
]


def __getattr__(name: str):
    if name in _LAZY:
        from importlib import import_module

        value = globals()[name] = getattr(import_module(f".{_LAZY[name]}", __name__), name)
        return value
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")


def __dir__() -> list[str]:
    return sorted({*globals(), *_LAZY})
