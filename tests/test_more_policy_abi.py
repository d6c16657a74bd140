"""C entry points of the layer norm: refusals before any HIP call and the size of
scratch memory (no GPU)."""

from __future__ import annotations

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
