"""What ``gbxcule_amd.rl`` gives without its operators' libraries."""

from __future__ import annotations

import subprocess
import sys
import textwrap

from .conftest import ROOT


def _python(code: str) -> subprocess.CompletedProcess:
    return subprocess.run([sys.executable, "-c", textwrap.dedent(code)], cwd=ROOT, capture_output=True, text=True, timeout=120)


def test_a_star_import_needs_neither_torch_nor_the_libraries():
    done = _python("""
        import sys
        sys.modules["torch"] = None  # an import raises
        from gbxcule_amd.rl import *
        assert RolloutBuffer and collect_rollout and packed_l1_distance
        assert not any(m in sys.modules for m in ("gbxcule_amd._torch_ops", "gbxcule_amd.rl.ops", "gbxcule_amd.rl.optim"))
    """)
    assert done.returncode == 0, done.stderr


def test_operators_are_found_by_name():
    import gbxcule_amd.rl as rl

    names = {"AdamW", "causal_conv", "causal_conv_step", "rms_norm", "rms_norm_fp8", "selective_scan", "selective_scan_step"}
    assert names <= set(dir(rl)) and set(rl.__all__) <= set(dir(rl))
