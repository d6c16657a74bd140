"""C entry points of the layer norm, the delta rule and sampling: refusals before
any HIP call and the size of scratch memory (no GPU)."""

from __future__ import annotations

import math

import pytest

from gbxcule_amd import _lib

P = 4096  # an address that no call here gets to use


def _bad(rc: int, text: bytes) -> None:
    assert rc == _lib.GBX_E_INVALID
    assert text in _lib.load().gbx_last_error()


def test_layer_norm_arguments():
    lib = _lib.load()
    call = lambda rows=1, dim=8, elem=0, x=P, weight=P, res=None, summed=None: lib.gbx_layer_norm(  # noqa: E731
        rows, dim, elem, 1e-5, x, dim, res, dim, weight, None, P, summed, None)  # fmt: skip
    assert call(rows=0) == 0
    _bad(call(rows=-1), b"row count")
    _bad(call(dim=0), b"channel count")
    _bad(call(dim=(1 << 20) + 1), b"channel count")
    _bad(call(elem=3), b"element type")
    _bad(call(x=None), b"NULL")
    _bad(call(weight=None), b"NULL")
    _bad(call(res=P), b"together")
    _bad(call(summed=P), b"together")
    grad = lambda rows=1, dy=P, work=P: lib.gbx_layer_norm_grad(rows, 8, 0, 1e-5, P, 8, dy, 8, None, 0, P, P, P, None, work, None)  # noqa: E731
    _bad(grad(dy=None), b"NULL")
    _bad(grad(work=None), b"NULL")
    _bad(grad(rows=0), b"no rows")
    assert lib.gbx_layer_norm_grad_work(-1, 8) == _lib.GBX_E_INVALID
    assert lib.gbx_layer_norm_grad_work(1, 8) == 16 and lib.gbx_layer_norm_grad_work(1 << 30, 8) >= 16


def _delta_in(**change):
    good = dict(steps=4, envs=2, heads=4, share=2, keys=16, values=24, elem=0, normalize=1, scale=0.25, q=P, k=P, v=P, gate=P, beta=P)
    return _lib.DeltaIn(**{**good, **change})


@pytest.mark.parametrize(
    "change, text",
    [(dict(steps=0), b"step count"), (dict(envs=0), b"env count"), (dict(heads=0), b"head count"),
     (dict(share=3), b"multiple"), (dict(share=0), b"multiple"), (dict(keys=0), b"keys"), (dict(keys=129), b"keys"),
     (dict(values=0), b"values"), (dict(values=129), b"values"), (dict(elem=3), b"element type"),
     (dict(envs=1 << 26, heads=64, share=1), b"out of range"), (dict(q=None), b"NULL"), (dict(beta=None), b"NULL")],
)  # fmt: skip
def test_delta_rule_arguments(change, text):
    lib = _lib.load()
    given = _delta_in(**change)
    _bad(lib.gbx_delta_rule(given, None, P, P, None, P, None), text)
    _bad(lib.gbx_delta_rule_grad(given, P, P, 8, 8, 8, P, P, P, P, P, P, None), text)
    _bad(lib.gbx_delta_rule_step(given, P, P, None), text)
    assert lib.gbx_delta_rule_work(given) == _lib.GBX_E_INVALID
    assert lib.gbx_delta_rule_grad_work(given) == _lib.GBX_E_INVALID


def test_delta_rule_outputs_and_work():
    lib = _lib.load()
    given = _delta_in()
    _bad(lib.gbx_delta_rule(given, None, None, P, None, P, None), b"NULL")
    _bad(lib.gbx_delta_rule(given, None, P, None, None, P, None), b"NULL")
    _bad(lib.gbx_delta_rule(None, None, P, P, None, P, None), b"NULL")
    _bad(lib.gbx_delta_rule_grad(given, None, P, 8, 8, 8, P, P, P, P, P, P, None), b"NULL")
    _bad(lib.gbx_delta_rule_grad(given, P, P, 8, 8, 8, P, P, P, P, None, P, None), b"NULL")
    _bad(lib.gbx_delta_rule_grad(given, P, P, 8, 8, 8, P, P, P, P, P, None, None), b"work")
    _bad(lib.gbx_delta_rule_step(given, P, P, None), b"steps")
    _bad(lib.gbx_delta_rule_step(_delta_in(steps=1), None, P, None), b"NULL")
    # two heads' gradients of the rows that they share are added in scratch memory
    assert lib.gbx_delta_rule_grad_work(given) >= 2 * 4 * 2 * 4 * 16
    assert lib.gbx_delta_rule_work(given) >= 0 and lib.gbx_delta_rule_grad_work(_delta_in(share=1)) >= 0


def _sample_in(**change):
    good = dict(rows=3, actions=8, elem=0, logits=P, stride=8, uniform=P, temperature=1.0, top_p=1.0, min_p=0.0)
    return _lib.SampleIn(**{**good, **change})


@pytest.mark.parametrize(
    "change, text",
    [(dict(rows=-1), b"row count"), (dict(actions=0), b"channel count"), (dict(actions=(1 << 20) + 1), b"channel count"),
     (dict(elem=5), b"element type"), (dict(logits=None), b"NULL"), (dict(uniform=None), b"NULL"),
     (dict(temperature=-1.0), b"temperature"), (dict(temperature=math.nan), b"temperature"), (dict(top_p=0.0), b"top_p"),
     (dict(min_p=2.0), b"min_p")],
)  # fmt: skip
def test_sample_arguments(change, text):
    lib = _lib.load()
    _bad(lib.gbx_sample_actions(_sample_in(**change), P, P, None), text)


def test_sample_outputs():
    lib = _lib.load()
    _bad(lib.gbx_sample_actions(None, P, P, None), b"NULL")
    _bad(lib.gbx_sample_actions(_sample_in(), None, P, None), b"NULL")
    _bad(lib.gbx_sample_actions(_sample_in(), P, None, None), b"NULL")
    assert lib.gbx_sample_actions(_sample_in(rows=0), None, None, None) == 0


def test_delta_rule_work_of_pieces():
    """Few heads and many steps go in pieces, whose states are in scratch memory; many heads need none."""
    lib = _lib.load()
    long = _delta_in(steps=8192, envs=1, heads=8, share=1)
    floats = lib.gbx_delta_rule_work(long)
    assert floats >= 3 * 8 * 16 * (24 + 16)
    _bad(lib.gbx_delta_rule(long, None, P, P, None, None, None), b"work")
    assert lib.gbx_delta_rule_work(_delta_in(steps=8192, envs=4096)) == 0
