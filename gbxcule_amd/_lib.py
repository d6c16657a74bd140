"""ctypes binding of ``libgbx_hip.so`` (the C ABI in ``include/gbx_hip.h``).

The library is loaded from ``gbxcule_amd/lib/``.  There is no fallback: if it
is missing or fails to load, every entry point raises.
"""

from __future__ import annotations

import ctypes
from pathlib import Path

LIB_PATH = Path(__file__).resolve().parent / "lib" / "libgbx_hip.so"

GBX_OK, GBX_E_INVALID, GBX_E_STATE, GBX_E_HIP, GBX_E_UNSUPPORTED = 0, -1, -2, -3, -4

FIELDS = (
    "pc", "sp", "a", "b", "c", "d", "e", "h", "l", "f",
    "instr_count", "cycle_count", "cycle_in_frame", "trap_flag", "trap_pc",
    "trap_opcode", "trap_kind", "actions", "joyp_select", "serial_len",
    "serial_overflow", "ime", "ime_delay", "halted", "div_counter",
    "timer_prev_in", "tima_reload_pending", "tima_reload_delay",
    "ppu_scanline_cycle", "ppu_ly", "ppu_window_line", "ppu_stat_prev",
)  # fmt: skip
FIELD_ID = {name: i for i, name in enumerate(FIELDS)}

BUF_MEM, BUF_PIX, BUF_PIX_PACKED, BUF_OBS, BUF_REWARD, BUF_ACTIONS, BUF_CART_RAM, BUF_FRAME_BG = range(8)
(
    INFO_NUM_ENVS,
    INFO_PADDED_ENVS,
    INFO_ROM_BANKS,
    INFO_ROM_BANK_MASK,
    INFO_RAM_BANKS,
    INFO_RAM_BYTES,
    INFO_MBC_KIND,
    INFO_OBS_DIM,
    INFO_CART_RAM_STRIDE,
    INFO_STEP_LANES,
    INFO_STEP_THREADS,
    INFO_STEP_WAVES,
) = range(12)

_vp, _i32, _i64, _f32, _f64 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float, ctypes.c_double


class ScanIn(ctypes.Structure):
    """``gbx_scan_in``."""

    _fields_ = [
        *((k, _i32) for k in ("steps", "envs", "dim", "groups", "states", "elem", "softplus")),
        *((k, _vp) for k in ("x", "dt", "z", "b", "c")),
        *((k, _i64) for k in ("x_step", "x_env", "dt_step", "dt_env", "z_step", "z_env")),
        *((k, _i64) for k in ("b_step", "b_env", "b_group", "c_step", "c_env", "c_group")),
        *((k, _vp) for k in ("a", "skip", "bias", "resets")),
    ]


class DeltaIn(ctypes.Structure):
    """``gbx_delta_in``."""

    _fields_ = [
        *((k, _i32) for k in ("steps", "envs", "heads", "share", "keys", "values", "elem", "normalize")),
        ("scale", _f32),
        *((k, _vp) for k in ("q", "k", "v")),
        *((f"{k}_{d}", _i64) for k in ("q", "k", "v") for d in ("step", "env", "head")),
        *((k, _vp) for k in ("gate", "beta")),
        *((k, _i64) for k in ("gate_step", "gate_env", "beta_step", "beta_env")),
        ("resets", _vp),
    ]


class SampleIn(ctypes.Structure):
    """``gbx_sample_in``."""

    _fields_ = [
        ("rows", _i64),
        *((k, _i32) for k in ("actions", "elem")),
        ("logits", _vp),
        ("stride", _i64),
        *((k, _vp) for k in ("uniform", "temperatures", "top_ps", "min_ps", "top_ks")),
        *((k, _f64) for k in ("temperature", "top_p", "min_p")),
        ("top_k", _i32),
    ]


class AdamwIn(ctypes.Structure):
    """``gbx_adamw_in``."""

    _fields_ = [
        *((k, _i32) for k in ("count", "elem", "grad_elem", "state_bits")),
        *((k, _vp) for k in ("params", "grads", "sizes", "starts", "exp_avg", "exp_avg_sq")),
        *((k, _vp) for k in ("exp_avg_scale", "exp_avg_sq_scale", "grad_scale")),
        *((k, _f64) for k in ("beta1", "beta2", "step_size", "inv_root2", "eps", "keep")),
        ("key", ctypes.c_uint32),
    ]


# Every symbol the header declares, with its ctypes signature.
_P64 = ctypes.POINTER(ctypes.c_int64)
SIGNATURES: dict[str, tuple[object, list[object]]] = {
    "gbx_last_error": (ctypes.c_char_p, []),
    "gbx_version": (ctypes.c_int, []),
    "gbx_create": (ctypes.c_int, [_i32, _vp, _i64, _vp, _i32, _i32, ctypes.POINTER(_vp)]),
    "gbx_destroy": (ctypes.c_int, [_vp]),
    "gbx_reset": (ctypes.c_int, [_vp, _vp]),
    "gbx_upload_actions": (ctypes.c_int, [_vp, _vp, _vp]),
    "gbx_step": (ctypes.c_int, [_vp, _vp, _i32, _i32, _i32, _vp]),
    "gbx_render": (ctypes.c_int, [_vp, _vp, _i64, _i32, _vp]),
    "gbx_render_bg_env0": (ctypes.c_int, [_vp, _vp, _vp]),
    "gbx_snapshot": (ctypes.c_int, [_vp, _i32, _i32, _vp]),
    "gbx_masked_reset": (ctypes.c_int, [_vp, _vp, _vp]),
    "gbx_gather_mem": (ctypes.c_int, [_vp, _vp, _i32, _vp, _vp]),
    "gbx_read_mem": (ctypes.c_int, [_vp, _i32, _i32, _i32, _i32, _vp, _vp]),
    "gbx_write_mem": (ctypes.c_int, [_vp, _i32, _i32, _i32, _i32, _vp, _vp]),
    "gbx_state_hash": (ctypes.c_int, [_vp, _vp, _vp]),
    "gbx_export_scalar": (ctypes.c_int, [_vp, _i32, _vp]),
    "gbx_export_scalars": (ctypes.c_int, [_vp, _i32, _vp]),
    "gbx_packed_l1": (ctypes.c_int, [_vp, _i64, _vp, _i64, _i64, _i64, ctypes.c_float, _vp, _vp]),
    "gbx_import_scalar": (ctypes.c_int, [_vp, _i32, _vp]),
    "gbx_export_mem": (ctypes.c_int, [_vp, _i32, _i32, _i32, _i32, _vp]),
    "gbx_import_mem": (ctypes.c_int, [_vp, _i32, _i32, _vp, _i32]),
    "gbx_export_cart_state": (ctypes.c_int, [_vp, _vp]),
    "gbx_import_cart_state": (ctypes.c_int, [_vp, _vp]),
    "gbx_export_cart_ram": (ctypes.c_int, [_vp, _i32, _i32, _vp]),
    "gbx_export_serial": (ctypes.c_int, [_vp, _vp]),
    "gbx_export_latches": (ctypes.c_int, [_vp, _vp]),
    "gbx_export_env": (ctypes.c_int, [_vp, _i32, _vp, _vp, _vp, _vp]),
    "gbx_export_env_noalloc": (ctypes.c_int, [_vp, _i32, _vp, _vp, _vp, _vp]),
    "gbx_import_env": (ctypes.c_int, [_vp, _i32, _vp, _vp, _vp, _vp, _vp]),
    "gbx_buffer": (ctypes.c_int, [_vp, _i32, ctypes.POINTER(_vp), _P64]),
    "gbx_info": (ctypes.c_int, [_vp, _i32, _P64]),
    "gbx_set_debug": (ctypes.c_int, [_vp, _i32, _i32, _i32, _i32]),
    "gbx_rms_norm": (ctypes.c_int, [_i64, _i32, _i32, _f32, _vp, _i64, _vp, _i64, _vp, _vp, _vp, _vp, _i32, _vp]),
    "gbx_rms_norm_grad_work": (_i64, [_i64, _i32]),
    "gbx_rms_norm_grad": (
        ctypes.c_int, [_i64, _i32, _i32, _f32, _vp, _i64, _vp, _i64, _vp, _i64, _vp, _vp, _vp, _vp, _vp]),
    "gbx_layer_norm": (ctypes.c_int, [_i64, _i32, _i32, _f32, _vp, _i64, _vp, _i64, *[_vp] * 5]),
    "gbx_layer_norm_grad_work": (_i64, [_i64, _i32]),
    "gbx_layer_norm_grad": (
        ctypes.c_int, [_i64, _i32, _i32, _f32, _vp, _i64, _vp, _i64, _vp, _i64, *[_vp] * 6]),
    "gbx_causal_conv": (ctypes.c_int, [*[_i32] * 6, _vp, _i64, _i64, *[_vp] * 7]),
    "gbx_causal_conv_grad_work": (_i64, [_i32] * 4),
    "gbx_causal_conv_grad": (ctypes.c_int, [*[_i32] * 6, _vp, _i64, _i64, *[_vp] * 5, _i64, _i64, *[_vp] * 5]),
    "gbx_causal_conv_step": (ctypes.c_int, [*[_i32] * 5, _vp, _i64, *[_vp] * 6]),
    "gbx_selective_scan_work": (_i64, [ctypes.POINTER(ScanIn)]),
    "gbx_selective_scan": (ctypes.c_int, [ctypes.POINTER(ScanIn), *[_vp] * 6]),
    "gbx_selective_scan_grad_work": (_i64, [ctypes.POINTER(ScanIn)]),
    "gbx_selective_scan_grad": (ctypes.c_int, [ctypes.POINTER(ScanIn), _vp, _vp, _i64, _i64, *[_vp] * 10]),
    "gbx_selective_scan_step": (ctypes.c_int, [ctypes.POINTER(ScanIn), *[_vp] * 3]),
    "gbx_delta_rule_saved": (_i64, [ctypes.POINTER(DeltaIn)]),
    "gbx_delta_rule_work": (_i64, [ctypes.POINTER(DeltaIn)]),
    "gbx_delta_rule": (ctypes.c_int, [ctypes.POINTER(DeltaIn), *[_vp] * 6]),
    "gbx_delta_rule_grad_work": (_i64, [ctypes.POINTER(DeltaIn)]),
    "gbx_delta_rule_grad": (ctypes.c_int, [ctypes.POINTER(DeltaIn), _vp, _vp, *[_i64] * 3, *[_vp] * 7]),
    "gbx_delta_rule_step": (ctypes.c_int, [ctypes.POINTER(DeltaIn), *[_vp] * 3]),
    "gbx_sample_actions": (ctypes.c_int, [ctypes.POINTER(SampleIn), *[_vp] * 3]),
    "gbx_adamw": (ctypes.c_int, [ctypes.POINTER(AdamwIn), _vp]),
}

_lib: ctypes.CDLL | None = None


class GbxError(RuntimeError):
    """A HIP runtime failure inside the library."""


def load() -> ctypes.CDLL:
    """Load the HIP library once; raise if it is absent."""
    global _lib
    if _lib is None:
        if not LIB_PATH.exists():
            raise RuntimeError(
                f"{LIB_PATH} is missing: build it with gbxcule_amd.build.build() "
                "(hipcc --offload-arch=gfx950)"
            )
        # torch bundles its own HIP runtime under the same soname as ROCm's.
        # Loading torch first makes the library bind to that runtime, so the
        # process holds one HIP runtime and device pointers are shared with
        # torch; loading the library first would put ROCm's runtime in place
        # and torch would then find no GPU.
        import torch  # noqa: F401

        lib = ctypes.CDLL(str(LIB_PATH))
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        _lib = lib
    return _lib


def check(rc: int) -> None:
    """Map a library status code to the reference's Python exception types."""
    if rc == GBX_OK:
        return
    msg = (load().gbx_last_error() or b"").decode(errors="replace")
    if rc == GBX_E_INVALID:
        raise ValueError(msg)
    if rc == GBX_E_STATE:
        raise RuntimeError(msg)
    if rc == GBX_E_UNSUPPORTED:
        raise ValueError(msg)
    raise GbxError(msg or f"libgbx_hip error {rc}")
