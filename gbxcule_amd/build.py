"""Build the HIP shared library ``gbxcule_amd/lib/libgbx_hip.so`` for gfx950 and
``gbxcule_amd/lib/gbx_torch.so``, the binding of its policy operators to torch
(where torch is installed: the library alone serves users of the C ABI).

``hipcc`` cross-compiles for gfx950 without a GPU present.  All HIP sources are
compiled with packed FP32 instructions disabled (``-packed-fp32-ops``).
"""

from __future__ import annotations

import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
LIB_DIR = PKG / "lib"
LIB_PATH = LIB_DIR / "libgbx_hip.so"
EXT_PATH = LIB_DIR / "gbx_torch.so"
EXT_SOURCE = "gbx_torch.cpp"
ARCH = os.environ.get("GBX_OFFLOAD_ARCH", "gfx950")
# -O2 with the iterative ILP machine scheduler: on the step kernel's hot
# loop this schedules the dependent loads earlier than -O3 with the default
# occupancy-first scheduler (same-box A/B: 16K-env CPU-step workload +2.4%,
# 131K-env banked cart +2.5%, RL rollout shape unchanged).
DEVICE_FLAGS = (
    "-O2",
    f"--offload-arch={ARCH}",
    "-std=c++17",
    "-mllvm",
    "-amdgpu-sched-strategy=iterative-ilp",
    "-Xclang",
    "-target-feature",
    "-Xclang",
    "-packed-fp32-ops",
)
# The policy operators: the default scheduler.  The other one leaves the
# gradient of the scan more spilled registers, and its register allocation
# crashes on the 8-bit AdamW kernel.
POLICY_SOURCES = ("gbx_norm.hip", "gbx_conv.hip", "gbx_scan.hip", "gbx_adamw.hip")
SOURCES = ("gbx_step.hip", "gbx_aux.hip", *POLICY_SOURCES, "gbx_api.hip")
POLICY_FLAGS = tuple(f for f in DEVICE_FLAGS if f != "-mllvm" and "sched-strategy" not in f)


def hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("hipcc not found; the HIP library cannot be built")


def _extension_command(out: Path) -> list[str]:
    """Host code only, against torch's headers and libraries: g++, or ROCm's
    compiler where there is none."""
    import torch
    from torch.utils import cpp_extension

    lib = Path(torch.__file__).resolve().parent / "lib"
    system = [*cpp_extension.include_paths("cuda"), sysconfig.get_paths()["include"]]
    return [
        shutil.which("g++") or str(Path(hipcc()).parent / "amdclang++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
        "-DTORCH_EXTENSION_NAME=gbx_torch", "-I", str(PKG.parent / "include"),
        *[flag for path in system for flag in ("-isystem", path)], str(CSRC / EXT_SOURCE), "-o", str(out),
        "-L", str(lib), "-L", str(LIB_DIR), "-lgbx_hip", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_hip", "-ltorch_python",
        "-Wl,-rpath,$ORIGIN",
    ]  # fmt: skip


def _run(commands: list[list[str]], verbose: bool) -> None:
    """The commands side by side; the first that fails is reported."""
    with ThreadPoolExecutor(max_workers=len(commands)) as pool:
        done = list(pool.map(lambda cmd: subprocess.run(cmd, capture_output=True, text=True), commands))
    for cmd, res in zip(commands, done):
        if verbose:
            print(" ".join(cmd), flush=True)
        if res.returncode != 0:
            sys.stderr.write(res.stdout + res.stderr)
            raise RuntimeError(f"build failed: {' '.join(cmd)}")


def build(verbose: bool = False) -> Path:
    """Compile every source and link both libraries (always rebuilds)."""
    LIB_DIR.mkdir(exist_ok=True)
    objects = [LIB_DIR / f"{Path(s).stem}.o" for s in SOURCES]
    include = ["-I", str(PKG.parent / "include")]
    _run(
        [
            [hipcc(), *(POLICY_FLAGS if s in POLICY_SOURCES else DEVICE_FLAGS), "-fPIC", *include, "-c", str(CSRC / s), "-o", str(o)]
            for s, o in zip(SOURCES, objects)
        ],
        verbose,
    )  # fmt: skip
    tmp = LIB_DIR / "libgbx_hip.so.tmp"
    _run([[hipcc(), f"--offload-arch={ARCH}", "-fPIC", "-shared", "-Wl,-soname,libgbx_hip.so", "-o", str(tmp), *map(str, objects)]], verbose)
    for o in objects:
        o.unlink()
    os.replace(tmp, LIB_PATH)
    if importlib.util.find_spec("torch") is None:
        print("torch is not installed: gbx_torch.so, which binds the policy operators to it, is not built", file=sys.stderr)
        return LIB_PATH
    tmp = LIB_DIR / "gbx_torch.so.tmp"
    _run([_extension_command(tmp)], verbose)
    os.replace(tmp, EXT_PATH)
    return LIB_PATH


if __name__ == "__main__":
    print(build(verbose=True))
