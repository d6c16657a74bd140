"""Layer norm against its plain 64-bit form: row lengths around every tile,
types, strides, rows far from zero, values that are not finite, gradients
against autograd and against differences, graphs, and refusals."""

from __future__ import annotations

import pytest
import torch

from . import _policy_ref as ref
from .conftest import require_gpu

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _gpu():
    require_gpu()


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape, dtype=F32, scale=1.0):
    return (torch.randn(shape, device="cuda", generator=gen) * scale).to(dtype)


def _plain(x, weight, bias, residual, eps, stream_type):
    """(y, s) in 64 bits; s is rounded to the stream's type, with the gradient of the sum."""
    s = x
    if residual is not None:
        s = x + residual
        s = s + (s.detach().to(stream_type).double() - s.detach())
    c = s - s.mean(-1, keepdim=True)
    y = c / torch.sqrt((c * c).mean(-1, keepdim=True) + eps) * weight
    return (y if bias is None else y + bias), s


def _roundings(dim):
    """Those of a sum over a row: a lane's own adds, the tree between lanes, a
    workgroup's wavefronts."""
    return 16 + 3 * dim.bit_length() + dim // 256


DIMS = [1, 2, 7, 8, 9, 64, 127, 128, 129, 256, 257, 511, 512, 520, 1000, 1024, 1025, 2048, 2049, 4096, 4100, 8192, 8193, 20000]


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("residual, bias", [(False, True), (True, False), (True, True)])
def test_forward_and_gradient(dim, dtype, residual, bias):
    from gbxcule_amd.rl import layer_norm

    gen = _gen(dim)
    rows = 5 if dim > 4000 else 37
    x, w = _randn(gen, rows, dim, dtype=dtype), 1.0 + _randn(gen, dim, scale=0.2)
    b = _randn(gen, dim, scale=0.3) if bias else None
    r = _randn(gen, rows, dim, dtype=dtype, scale=2.0) if residual else None
    dy, ds = _randn(gen, rows, dim, dtype=dtype), _randn(gen, rows, dim, dtype=dtype)
    x, w, b, r = (None if t is None else t.requires_grad_() for t in (x, w, b, r))
    leaves = [t for t in (x, w, b, r) if t is not None]
    eps = 0.5 if dim == 1 else 1e-5  # one channel is its own mean: nothing but rounding would be divided
    out = layer_norm(x, w, b, r, eps=eps)
    wx, ww, wb, wr = (ref.f64(t) for t in (x, w, b, r))
    y, s = _plain(wx, ww, wb, wr, eps, dtype)
    n = _roundings(dim)
    # the mean's own roundings, of values up to 4 times the spread, go on through y and the three means of the gradient
    if residual:
        ref.check(out[0], y, 2 * n, "y")
        assert torch.equal(out[1].detach().cpu().double(), s.detach())
        got = torch.autograd.grad(out, leaves, [dy, ds])
        want = torch.autograd.grad([y, s], [t for t in (wx, ww, wb, wr) if t is not None], [ref.f64(dy), ref.f64(ds)])
        with torch.no_grad():
            again = layer_norm(x, w, b, r, eps=eps)
        assert torch.equal(again[0], out[0]) and torch.equal(again[1], out[1])
    else:
        ref.check(out, y, 2 * n, "y")
        got = torch.autograd.grad(out, leaves, dy)
        want = torch.autograd.grad(y, [t for t in (wx, ww, wb) if t is not None], ref.f64(dy))
    names = [k for k, t in zip(("x", "weight", "bias", "residual"), (x, w, b, r)) if t is not None]
    if dim == 1:  # 64 bits give zeros, of which the largest value is no scale
        assert not got[0].float().any() or residual
        return
    for g, v, name in zip(got, want, names):
        if dim == 2 and name in ("x", "residual"):
            # c is plus and minus half a difference d, and r nearly 2 / d, so r * (g - mean(g) - c r^2 mean(g c)) is next to
            # nothing while its terms are r |g|.  What is left is their rounding: r |g| half steps each, and those of c,
            # half a step of |s|, which count r |s| times as much in c r.
            r = 1 / torch.sqrt(s.detach().var(-1, unbiased=False, keepdim=True) + eps)
            term = r * (ref.f64(dy) * ww.detach()).abs().amax(-1, keepdim=True) * (1 + r * s.detach().abs().amax(-1, keepdim=True))
            off = (g.cpu().double() - v).abs()
            assert bool((off <= n * 2.0**-23 * term + ref.UNIT[dtype] * v.abs() + ref.FLOOR[dtype]).all())
            continue
        ref.check(g, v, 4 * n + rows, f"gradient of {name}")


def test_rows_far_from_zero():
    """Means of 1,000 times the spread: the squares are of what is left when the mean is gone."""
    from gbxcule_amd.rl import layer_norm

    gen = _gen(5)
    x = _randn(gen, 11, 700) + 1000.0
    w, b = torch.ones(700, device="cuda"), torch.zeros(700, device="cuda")
    y, _ = _plain(ref.f64(x), ref.f64(w), ref.f64(b), None, 1e-5, F32)
    # the mean is off by at most as many half steps of 1,000 as it has roundings; so is every centred value
    atol = _roundings(700) * 2.0**-24 * 1010.0
    assert float((layer_norm(x, w, b).cpu().double() - y).abs().max()) < 2 * atol


def test_strides_types_and_special_rows():
    from gbxcule_amd.rl import layer_norm

    gen = _gen(3)
    base = _randn(gen, 6, 5, 300, dtype=BF16)
    w, b = 1.0 + _randn(gen, 100, scale=0.1), _randn(gen, 100)
    for x in (base[..., 100:200], base[..., 1:101], base[::2, 1:4, 7:107], base[..., ::3], base[:, :1, :100].expand(6, 5, 100)):
        y, _ = _plain(ref.f64(x), ref.f64(w), ref.f64(b), None, 1e-5, BF16)
        ref.check(layer_norm(x, w, b), y, 64, str(x.stride()))
    one = base[0, 0, :100]
    assert layer_norm(one, w, b).shape == (100,) and torch.equal(layer_norm(one, w, b), layer_norm(base[0, :1, :100], w, b)[0])
    x = _randn(gen, 4, 512)
    x[1, 7], x[2, 9] = float("nan"), float("inf")
    y = layer_norm(x, torch.ones(512, device="cuda"))
    assert torch.isnan(y[1:3]).all() and torch.isfinite(y[[0, 3]]).all()
    assert not layer_norm(torch.full((3, 512), 7.0, device="cuda"), torch.ones(512, device="cuda")).any()  # a row of equals
    # parameters in the stream's type get their gradients in that type
    wb, bb = w.to(BF16).requires_grad_(), b.to(BF16).requires_grad_()
    gw, gb = torch.autograd.grad(layer_norm(base[0, :, :100], wb, bb).float().sum(), [wb, bb])
    assert gw.dtype is BF16 and gb.dtype is BF16 and torch.equal(gb.float(), torch.full((100,), 5.0, device="cuda"))


def test_no_rows_and_the_sum_alone():
    from gbxcule_amd.rl import layer_norm

    gen = _gen(8)
    w, b = torch.ones(64, device="cuda", requires_grad=True), torch.zeros(64, device="cuda", requires_grad=True)
    x = torch.zeros(0, 3, 64, device="cuda", requires_grad=True)
    gx, gw, gb = torch.autograd.grad(layer_norm(x, w, b).sum(), [x, w, b])
    assert gx.shape == x.shape and not gw.any() and not gb.any()
    x, r = _randn(gen, 5, 64).requires_grad_(), _randn(gen, 5, 64).requires_grad_()
    _, s = layer_norm(x, w, b, r)
    gx, gr, gw, gb = torch.autograd.grad(s.sum(), [x, r, w, b])
    assert torch.equal(gx, torch.ones_like(gx)) and torch.equal(gr, gx) and not gw.any() and not gb.any()
    y, _ = layer_norm(x, w, b, r)  # y alone: no gradient comes in for the sum
    (gx,) = torch.autograd.grad(y.sum(), x)
    assert torch.isfinite(gx).all()


def test_gradient_against_differences():
    from gbxcule_amd.rl import layer_norm

    gen = _gen(9)
    tensors = [_randn(gen, 6, 45), 1.0 + _randn(gen, 45, scale=0.3), _randn(gen, 45), _randn(gen, 6, 45)]
    toward = [_randn(gen, *t.shape) for t in tensors]
    wy, ws = _randn(gen, 6, 45).double(), _randn(gen, 6, 45).double()

    def loss(leaves):
        y, s = layer_norm(*leaves)
        return (y.double() * wy).sum() + (s.double() * ws).sum()

    leaves = [t.requires_grad_() for t in tensors]
    slope = sum(float((g * d).double().sum()) for g, d in zip(torch.autograd.grad(loss(leaves), leaves), toward))
    step = 2.0**-8
    with torch.no_grad():
        up, down = (float(loss([t + sign * step * d for t, d in zip(tensors, toward)])) for sign in (1, -1))
    # each side: 540 values of up to 5 with half a dozen roundings, 2^-24 each, of random sign; over the
    # distance; and the third derivative, about the size of the first, times a sixth of the step's square
    assert abs((up - down) / (2 * step) - slope) < 2.0**-24 * 6 * 5 * 540**0.5 * 3 / step + abs(slope) * step**2 + 1e-3


def test_more_rows_than_a_launch_has_turns_for():
    """Each of the gradient's workgroups takes several turns of rows; twice, bit for bit."""
    from gbxcule_amd.rl import layer_norm

    gen = _gen(13)
    rows, dim = 1024 * 16 + 5, 96
    x, w, b = _randn(gen, rows, dim).requires_grad_(), torch.ones(dim, device="cuda", requires_grad=True), torch.zeros(dim, device="cuda", requires_grad=True)
    dy = _randn(gen, rows, dim)
    got = [torch.autograd.grad(layer_norm(x, w, b), [x, w, b], dy) for _ in range(2)]
    assert all(torch.equal(p, q) for p, q in zip(*got))
    wide = [ref.f64(t) for t in (x, w, b)]
    y, _ = _plain(*wide, None, 1e-5, F32)
    want = torch.autograd.grad(y, wide, ref.f64(dy))
    for g, v, name in zip(got[0], want, ("x", "weight", "bias")):
        ref.check(g, v, 100, f"gradient of {name}")


def test_another_stream_and_a_graph():
    from gbxcule_amd.rl import layer_norm

    gen = _gen(21)
    x, r, w, b = _randn(gen, 300, 250, dtype=BF16), _randn(gen, 300, 250, dtype=BF16), torch.ones(250, device="cuda"), _randn(gen, 250)
    want = layer_norm(x, w, b, r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layer_norm(x, w, b, r)
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer_norm(x, w, b, r)
    for k in range(3):
        x.copy_(_randn(gen, 300, 250, dtype=BF16))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, layer_norm(x, w, b, r)))


def test_refusals():
    import torch.autograd.forward_ad as fwad

    from gbxcule_amd.rl import layer_norm

    x, w = torch.randn(4, 8, device="cuda"), torch.ones(8, device="cuda")
    for bad in (
        lambda: layer_norm(x.cpu(), w),
        lambda: layer_norm(x.double(), w),
        lambda: layer_norm(x, w[:7]),
        lambda: layer_norm(x, w, w[:7]),
        lambda: layer_norm(x, w, w.cpu()),
        lambda: layer_norm(x, w, torch.ones(8, device="cuda", dtype=torch.int32)),
        lambda: layer_norm(x, w, w, x[:3]),
        lambda: layer_norm(x, w, w, x.half()),
        lambda: layer_norm(torch.zeros(4, 0, device="cuda"), w[:0]),
        lambda: layer_norm(torch.zeros((), device="cuda"), w),
    ):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        layer_norm(x, [1.0] * 8)
    xg = x.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(layer_norm(xg, w, w).sum(), xg, create_graph=True)
    with fwad.dual_level(), pytest.raises(NotImplementedError):
        layer_norm(fwad.make_dual(x, torch.ones_like(x)), w)
