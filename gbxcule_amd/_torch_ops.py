"""Loader of ``gbx_torch``, the torch binding of the policy operators
(``csrc/gbx_torch.cpp``).  There is no fallback: if it is missing or fails to
load, every operator raises."""

from __future__ import annotations

from importlib.machinery import ExtensionFileLoader
from importlib.util import module_from_spec, spec_from_loader
from pathlib import Path

from . import _lib

EXT_PATH = Path(__file__).resolve().parent / "lib" / "gbx_torch.so"


def _load():
    if not EXT_PATH.exists():
        raise RuntimeError(f"{EXT_PATH} is missing: build it with gbxcule_amd.build.build()")
    _lib.load()  # after torch, whose HIP runtime both bind to
    loader = ExtensionFileLoader("gbx_torch", str(EXT_PATH))
    module = module_from_spec(spec_from_loader("gbx_torch", loader))
    loader.exec_module(module)
    return module


ext = _load()
