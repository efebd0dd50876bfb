"""GPU tests of layer norm (ops.layer_norm, ops.layer_norm_backward) against a
plain implementation in 64 bits.

Tolerances.  A row's sums are chains of at most 16 values a thread, then trees
of at most 10 steps: their error is below 29 * 2^-24 of the terms' sum.  The
centred values' mean is taken off, so xhat is off by 29 * 2^-24 through the
mean, by half of that relatively through the variance, by 2 units in the last
place (2^-22) through the reciprocal root and by a few roundings: below
40 * 2^-24 (1 + |xhat|).  dx adds two more such sums over a and a * xhat, dweight
and dbias a chain over a block's rows and a tree over the blocks: 96 * 2^-24 of
the terms' sum.  What is stored in bfloat16 is off by half a step more.
"""
from __future__ import annotations

import pytest
import torch

from moonxi_net_b200 import _lib, ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16


def _half_step(t):
    return torch.finfo(t).eps / 2 if t is not F32 else 0.0


def _problem(rows, cols, dtype, seed=0, offset=0.0):
    g = torch.Generator("cuda").manual_seed(seed)

    def randn(*s):
        return torch.randn(*s, device="cuda", generator=g)
    x = (randn(rows, cols) * (1 + 3 * torch.rand(rows, 1, device="cuda", generator=g)) + offset)
    return x.to(dtype), (1 + randn(cols)), randn(cols), randn(rows, cols).to(dtype)


def _reference(x, w, b, dy, eps):
    x, dy = x.double(), dy.double()
    w = torch.ones(x.shape[1], device=x.device, dtype=torch.double) if w is None else w.double()
    b = torch.zeros_like(w) if b is None else b.double()
    mean = x.mean(1, keepdim=True)
    var = ((x - mean) ** 2).mean(1, keepdim=True)
    rstd = (var + eps).rsqrt()
    xh = (x - mean) * rstd
    a = dy * w
    c1, c2 = a.mean(1, keepdim=True), (a * xh).mean(1, keepdim=True)
    ref = {"y": xh * w + b, "dx": rstd * (a - c1 - xh * c2), "dw": (dy * xh).sum(0), "db": dy.sum(0)}
    m1, m2 = a.abs().mean(1, keepdim=True), (a * xh).abs().mean(1, keepdim=True)
    tol = {"y": 40 * U * ((1 + xh.abs()) * w.abs() + b.abs()),
           "dx": 96 * U * rstd * (a.abs() + m1 + (1 + xh.abs()) * (m2 + m1)),
           "dw": 96 * U * (dy.abs() * (1 + xh.abs())).sum(0), "db": 96 * U * dy.abs().sum(0)}
    return ref, tol


def _check(name, got, ref, tol):
    lim = tol + _half_step(got.dtype) * ref.abs()
    bad = (got.double() - ref).abs() > lim
    assert not bad.any(), (name, int(bad.sum()), float(((got.double() - ref).abs() / lim).max()))


def _all(x, w, b, dy, eps=1e-5, **kw):
    y, mean, rstd = ops.layer_norm(x, w, b, eps, stats=True, **kw)
    dx, dw, db = ops.layer_norm_backward(dy, x, w, mean, rstd, **kw)
    return {"y": y, "dx": dx, "dw": dw, "db": db}


# the sizes around each kernel's limits: a warp's row, a block's, long rows
SIZES = [(1, 1), (1, 8), (1025, 40), (1100, 300), (1024, 511), (1030, 520), (1200, 1000), (3, 7), (5, 33), (130, 256), (77, 257), (9, 512), (1000, 513), (4, 1024),
         (300, 1500), (600, 2048), (333, 2056), (700, 4100), (40, 8192), (19, 10000), (9, 16384),
         (5, 16385), (70, 20000), (2000, 64)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,cols", SIZES)
def test_against_64_bits(cuda_device, rows, cols, dtype):
    x, w, b, dy = _problem(rows, cols, dtype, rows * 7 + cols)
    ref, tol = _reference(x, w, b, dy, 1e-5)
    got = _all(x, w, b, dy)
    for k in ref:
        _check(k, got[k], ref[k], tol[k])
    again = _all(x, w, b, dy)
    assert all(torch.equal(got[k], again[k]) for k in got)  # a fixed order of sums


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_without_weight_and_bias(cuda_device, dtype):
    x, _, _, dy = _problem(37, 300, dtype)
    ref, tol = _reference(x, None, None, dy, 1e-5)
    got = _all(x, None, None, dy)
    for k in ref:
        _check(k, got[k], ref[k], tol[k])


@pytest.mark.parametrize("offset", [1e2, 1e4])
def test_a_mean_far_above_the_deviation(cuda_device, offset):
    """x itself is rounded to float32; the norm of what is stored is not lost."""
    x, w, b, dy = _problem(64, 1000, F32, 3, offset)
    ref, tol = _reference(x, w, b, dy, 1e-5)
    # the mean is held in float32: the saved mean costs the backward pass
    # 2^-24 of it, in units of the deviation
    slack = offset * U / x.double().std(1, keepdim=True)
    y, mean, rstd = ops.layer_norm(x, w, b, stats=True)
    _check("y", y, ref["y"], tol["y"])
    dx, dw, db = ops.layer_norm_backward(dy, x, w, mean, rstd)
    a = (dy * w).double().abs()
    r = rstd.double().unsqueeze(1)
    _check("dx", dx, ref["dx"], tol["dx"] + 4 * r * slack * (a.mean(1, keepdim=True) * 2 + a))
    _check("dw", dw, ref["dw"], tol["dw"] + (dy.double().abs() * 2 * slack).sum(0))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("start,cols,pitch", [(0, 256, 300), (8, 512, 1032), (3, 200, 211), (1, 4096, 4100)])
def test_row_strides(cuda_device, dtype, start, cols, pitch):
    """Rows inside a wider matrix: the values beside them stay as they were."""
    x, w, b, dy = _problem(50, cols, dtype)
    ref, tol = _reference(x, w, b, dy, 1e-5)
    bufs = [torch.full((50, pitch), 7.0, device="cuda", dtype=dtype) for _ in range(4)]
    xs, dys, ys, dxs = (t[:, start:start + cols] for t in bufs)
    xs.copy_(x)
    dys.copy_(dy)
    y, mean, rstd = ops.layer_norm(xs, w, b, stats=True, out=ys)
    dx, dw, db = ops.layer_norm_backward(dys, xs, w, mean, rstd, dx=dxs)
    for k, g in (("y", y), ("dx", dx), ("dw", dw), ("db", db)):
        _check(k, g, ref[k], tol[k])
    for t in bufs:
        rest = torch.cat((t[:, :start], t[:, start + cols:]), 1)
        assert (rest == 7.0).all()


def test_leading_dimensions_and_empty(cuda_device):
    x, w, b, dy = _problem(24, 96, BF16)
    y = ops.layer_norm(x, w, b)[0]
    y3 = ops.layer_norm(x.view(2, 3, 4, 96), w, b)[0]
    assert y3.shape == (2, 3, 4, 96) and torch.equal(y3.view(24, 96), y)
    none = torch.empty(0, 96, device="cuda", dtype=BF16)
    y, mean, rstd = ops.layer_norm(none, w, b, stats=True)
    assert y.shape == (0, 96) and mean.numel() == 0
    dx, dw, db = ops.layer_norm_backward(none, none, w, mean, rstd)
    assert dx.shape == (0, 96) and (dw == 0).all() and (db == 0).all()


def test_rows_are_independent_of_what_is_not_finite(cuda_device):
    x, w, b, dy = _problem(9, 700, F32)
    good = _all(x, w, b, dy)
    x2 = x.clone()
    x2[3, 5] = float("inf")
    x2[6, 0] = float("nan")
    y, mean, rstd = ops.layer_norm(x2, w, b, stats=True)
    keep = [0, 1, 2, 4, 5, 7, 8]
    assert torch.equal(y[keep], good["y"][keep])
    assert y[3].isnan().all() and y[6].isnan().all()
    dx = ops.layer_norm_backward(dy, x2, w, mean, rstd)[0]
    assert torch.equal(dx[keep], good["dx"][keep]) and dx[6].isnan().all()


def test_constant_row(cuda_device):
    """No deviation: eps alone; y is the bias."""
    x = torch.full((2, 512), 3.25, device="cuda")
    w, b = torch.full((512,), 2.0, device="cuda"), torch.randn(512, device="cuda")
    y, mean, rstd = ops.layer_norm(x, w, b, eps=1e-6, stats=True)
    assert torch.equal(y, b.expand(2, 512))
    assert torch.allclose(mean, torch.full_like(mean, 3.25)) and torch.allclose(
        rstd, torch.full_like(rstd, 1e3), rtol=4 * 2.0 ** -22)


def test_gradient_against_differences(cuda_device):
    """dx, dweight and dbias against a central difference of sum(dy * y) along a
    random direction, in 64 bits on the plain form."""
    x, w, b, dy = _problem(6, 40, F32, 5)
    got = _all(x, w, b, dy)
    g = torch.Generator("cuda").manual_seed(1)
    dirs = [torch.randn(t.shape, device="cuda", generator=g, dtype=torch.double) for t in (x, w, b)]

    def loss(h):
        xx, ww, bb = (t.double() + h * d for t, d in zip((x, w, b), dirs))
        return (_reference(xx, ww, bb, dy, 1e-5)[0]["y"] * dy.double()).sum()
    h = 1e-5
    diff = float((loss(h) - loss(-h)) / (2 * h))
    form = sum(float((got[k].double() * d).sum()) for k, d in zip(("dx", "dw", "db"), dirs))
    # h^2 of the difference's own error, and the gradients' float32
    scale = sum(float((got[k].double() * d).abs().sum()) for k, d in zip(("dx", "dw", "db"), dirs))
    assert abs(diff - form) <= scale * (200 * U + 1e-7)


def test_streams_and_capture(cuda_device):
    x, w, b, dy = _problem(300, 1000, BF16)
    want = _all(x, w, b, dy)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = [_all(x, w, b, dy, stream=s) for s in streams for _ in range(4)]
    torch.cuda.synchronize()
    assert all(torch.equal(want[k], t[k]) for t in got for k in want)
    graph = torch.cuda.CUDAGraph()
    xs = x.clone()
    with torch.cuda.graph(graph):
        out = _all(xs, w, b, dy)
    for seed in (1, 2):
        x2 = _problem(300, 1000, BF16, seed)[0]
        xs.copy_(x2)
        graph.replay()
        want = _all(x2, w, b, dy)
        assert all(torch.equal(want[k], out[k]) for k in want)


def test_refusals(cuda_device):
    x, w, b, dy = _problem(8, 64, F32)
    _, mean, rstd = ops.layer_norm(x, stats=True)
    with pytest.raises(TypeError):
        ops.layer_norm(x.half())
    with pytest.raises(TypeError):
        ops.layer_norm(x, w.to(BF16))
    with pytest.raises(ValueError):
        ops.layer_norm(x, w[:32])
    with pytest.raises(ValueError):
        ops.layer_norm(x, w, b[:1])
    with pytest.raises(ValueError):
        ops.layer_norm(x.t())
    with pytest.raises(ValueError):
        ops.layer_norm(x, w, b, out=torch.empty(8, 64, device="cuda", dtype=BF16))
    with pytest.raises(ValueError):
        ops.layer_norm_backward(dy[:4], x, w, mean, rstd)
    with pytest.raises(ValueError):
        ops.layer_norm_backward(dy, x, w, mean[:4], rstd)
    with pytest.raises(_lib.MXError, match="invalid argument"):
        ops.layer_norm(x, w, b, eps=-1.0)
    with pytest.raises(_lib.MXError, match="invalid argument"):
        ops.layer_norm(x, w, b, eps=float("nan"))
    L, h, p = _lib.lib(), ops.context(0), x.data_ptr()
    bad = _lib.MX_ERR_INVALID
    assert L.mx_layer_norm_fwd(h, 2, p, 64, None, None, p, 64, None, None, 8, 64, 1e-5, None) == bad
    assert L.mx_layer_norm_fwd(h, 0, p, 63, None, None, p, 64, None, None, 8, 64, 1e-5, None) == bad
    assert L.mx_layer_norm_fwd(h, 0, None, 64, None, None, p, 64, None, None, 8, 64, 1e-5, None) == bad
    assert L.mx_layer_norm_fwd(h, 0, p, 64, None, None, p, 64, None, None, -1, 64, 1e-5, None) == bad
    assert L.mx_layer_norm_bwd_scratch_bytes(h, 8, 64) == 0
    x, w, b, dy = _problem(1100, 64, F32)
    p = x.data_ptr()
    _, mean, rstd = ops.layer_norm(x, stats=True)
    need = L.mx_layer_norm_bwd_scratch_bytes(h, 1100, 64)
    args = (h, 0, dy.data_ptr(), 64, p, 64, None, mean.data_ptr(), rstd.data_ptr(), None, 0,
            w.data_ptr(), None, 1100, 64)
    assert L.mx_layer_norm_bwd(*args, p, need - 1, None) == bad
    assert L.mx_layer_norm_bwd(*args, None, need, None) == bad


def test_shared_memory_and_sizes_are_refused(cuda_device):
    x, w, b, dy = _problem(8, 64, F32)
    _, mean, rstd = ops.layer_norm(x, stats=True)
    with pytest.raises(ValueError, match="share memory"):
        ops.layer_norm(x, w, b, out=x)
    with pytest.raises(ValueError, match="share memory"):
        ops.layer_norm_backward(dy, x, w, mean, rstd, dx=dy)
    with pytest.raises(ValueError, match="share memory"):
        ops.layer_norm_backward(dy, x, w, mean, rstd, dweight=w)
    one = torch.empty(64, device="cuda")
    with pytest.raises(ValueError, match="share memory"):
        ops.layer_norm_backward(dy, x, w, mean, rstd, dweight=one, dbias=one)
    # halves of the same rows do not
    both = torch.randn(8, 128, device="cuda")
    ref = ops.layer_norm(both[:, 64:].contiguous(), w, b)[0]
    ops.layer_norm(both[:, 64:], w, b, out=both[:, :64])
    assert torch.equal(both[:, :64], ref)
    L, h, p = _lib.lib(), ops.context(0), x.data_ptr()
    top = 2 ** 31 - 1
    for rows, cols in ((1, top), (top, 1)):
        assert L.mx_layer_norm_fwd(h, 0, p, cols, None, None, p, cols, None, None, rows, cols, 1e-5,
                                   None) == _lib.MX_ERR_UNSUPPORTED
        assert L.mx_layer_norm_bwd_scratch_bytes(h, rows, cols) == 0
