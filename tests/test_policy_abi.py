"""The policy operators' C entry points refuse bad arguments before any HIP
call, and say how much scratch memory good ones need (no GPU)."""

from __future__ import annotations

import ctypes

import pytest

from gbxcule_amd import _lib

P = 4096  # an address that no call here gets to use


def _bad(rc: int, text: bytes) -> None:
    assert rc == _lib.GBX_E_INVALID
    assert text in _lib.load().gbx_last_error()


def test_norm_arguments():
    lib = _lib.load()
    call = lambda rows=1, dim=8, elem=0, x=P, res=None, summed=None, group=0: lib.gbx_rms_norm(  # noqa: E731
        rows, dim, elem, 1e-6, x, dim, res, dim, P, P, summed, None, group, None)  # fmt: skip
    assert call(rows=0) == 0
    _bad(call(rows=-1), b"row count")
    _bad(call(dim=0), b"channel count")
    _bad(call(dim=(1 << 20) + 1), b"channel count")
    _bad(call(elem=3), b"element type")
    _bad(call(x=None), b"NULL")
    _bad(call(res=P), b"together")
    _bad(call(group=64), b"group")
    _bad(lib.gbx_rms_norm_grad(1, 8, 0, 1e-6, P, 8, P, 8, None, 0, P, P, P, None, None), b"NULL")
    _bad(lib.gbx_rms_norm_grad(0, 8, 0, 1e-6, P, 8, P, 8, None, 0, P, P, P, P, None), b"no rows")
    assert lib.gbx_rms_norm_grad_work(-1, 8) == _lib.GBX_E_INVALID
    assert lib.gbx_rms_norm_grad_work(1, 8) == 8 and lib.gbx_rms_norm_grad_work(1 << 30, 8) >= 8


def test_conv_arguments():
    lib = _lib.load()
    call = lambda steps=1, envs=1, dim=8, width=4, elem=0, x=P: lib.gbx_causal_conv(  # noqa: E731
        steps, envs, dim, width, elem, 1, x, dim, dim, P, None, None, None, P, P, None)  # fmt: skip
    _bad(call(steps=0), b"step count")
    _bad(call(envs=0), b"env count")
    _bad(call(dim=-3), b"channel count")
    _bad(call(width=1), b"width")
    _bad(call(width=5), b"width")
    _bad(call(elem=-1), b"element type")
    _bad(call(x=None), b"NULL")
    _bad(lib.gbx_causal_conv_step(1, 8, 4, 0, 1, P, 8, P, None, None, None, P, None), b"NULL")
    _bad(lib.gbx_causal_conv_grad(1, 1, 8, 4, 0, 1, P, 8, 8, P, None, None, None, P, 8, 8, P, P, None, None, None), b"NULL")
    assert lib.gbx_causal_conv_grad_work(1, 1, 8, 9) == _lib.GBX_E_INVALID
    assert lib.gbx_causal_conv_grad_work(128, 16, 64, 4) >= 2 * 5 * 64


def _scan_in(**change):
    good = dict(steps=4, envs=2, dim=8, groups=2, states=16, elem=0, softplus=1, x=P, dt=P, b=P, c=P, a=P)
    return _lib.ScanIn(**{**good, **change})


@pytest.mark.parametrize(
    "change, text",
    [(dict(steps=0), b"step count"), (dict(envs=-1), b"env count"), (dict(dim=0), b"channel count"),
     (dict(groups=3), b"multiple"), (dict(groups=0), b"multiple"), (dict(states=0), b"states"),
     (dict(states=33), b"states"), (dict(elem=9), b"element type"), (dict(x=None), b"NULL"), (dict(a=None), b"NULL")],
)  # fmt: skip
def test_scan_arguments(change, text):
    lib = _lib.load()
    given = _scan_in(**change)
    _bad(lib.gbx_selective_scan(given, None, P, P, None, P, None), text)
    _bad(lib.gbx_selective_scan_grad(given, P, P, 8, 8, P, P, None, P, P, P, None, None, P, None), text)
    _bad(lib.gbx_selective_scan_step(given, P, P, None), text)
    assert lib.gbx_selective_scan_work(given) == _lib.GBX_E_INVALID
    assert lib.gbx_selective_scan_grad_work(given) == _lib.GBX_E_INVALID


def test_scan_outputs_and_work():
    lib = _lib.load()
    given = _scan_in()
    _bad(lib.gbx_selective_scan(given, None, None, P, None, P, None), b"NULL")
    _bad(lib.gbx_selective_scan_grad(given, P, P, 8, 8, P, P, P, P, P, P, None, None, P, None), b"together")
    _bad(lib.gbx_selective_scan_step(given, P, P, None), b"steps")
    _bad(lib.gbx_selective_scan(None, None, P, P, None, P, None), b"NULL")
    many = _scan_in(steps=1000, envs=1)
    assert lib.gbx_selective_scan_work(many) > 0  # one row is cut along the steps
    _bad(lib.gbx_selective_scan(many, None, P, P, None, None, None), b"work")
    assert lib.gbx_selective_scan_work(_scan_in(envs=100_000)) == 0
    assert lib.gbx_selective_scan_grad_work(given) > 0


def test_adamw_arguments():
    lib = _lib.load()
    one = lambda v, kind=ctypes.c_uint64: ctypes.cast((kind * 1)(v), ctypes.c_void_p)  # noqa: E731

    def call(**change):
        good = dict(count=1, elem=0, grad_elem=0, state_bits=32, params=one(P), grads=one(P), sizes=one(5), starts=one(0),
                    exp_avg=P, exp_avg_sq=P)  # fmt: skip
        return lib.gbx_adamw(_lib.AdamwIn(**{**good, **change}), None)

    assert call(count=0) == 0
    _bad(call(count=-1), b"negative")
    _bad(call(elem=4), b"types")
    _bad(call(elem=1, grad_elem=2), b"types")
    _bad(call(state_bits=16), b"state_bits")
    _bad(call(params=None), b"NULL")
    _bad(call(state_bits=8), b"NULL")
    _bad(call(sizes=one(-1, ctypes.c_int64)), b"size")
    _bad(call(starts=one(100)), b"256")
    _bad(call(params=one(0)), b"NULL")
