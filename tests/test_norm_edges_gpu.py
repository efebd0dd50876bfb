"""More GPU tests of layer norm, with the reference and tolerances of
test_norm_gpu.py."""
from __future__ import annotations

import pytest
import torch

from moonxi_net_b200 import ops
from test_norm_gpu import _check, _problem, _reference

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
# one for each backward kernel: the small one, a warp's rows, a block's, long rows
SHAPES = [(64, 100), (1100, 200), (1025, 300), (1030, 520), (600, 1100), (333, 2056), (40, 4104), (9, 8200)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_constant_rows(cuda_device, rows, cols, dtype):
    """Rows without deviation (padding, say) have no normalised part, however
    large their value is against 1 / rstd = sqrt(eps): x - mean comes before the
    product with rstd.  (The mean is given exactly here: what its own rounding
    costs is another test's.)"""
    _, w, b, dy = _problem(rows, cols, dtype, 1)
    for value, eps in ((1000.0, 1e-5), (2.0 ** 30, 1e-6), (2.0 ** 112, 1e-12)):
        x = torch.full((rows, cols), value, device="cuda", dtype=dtype)
        x[::2] = -value / 2
        ref, tol = _reference(x, w, b, dy, eps)
        rstd = torch.full((rows,), eps ** -0.5, device="cuda")
        dx, dw, db = ops.layer_norm_backward(dy, x, w, x[:, 0].float().contiguous(), rstd)
        assert (dw == 0).all(), value
        for k, got in (("dx", dx), ("db", db)):
            _check((k, value), got, ref[k], tol[k])


@pytest.mark.parametrize("rows,cols", SHAPES)
def test_a_mean_far_above_the_deviation(cuda_device, rows, cols):
    """The backward pass of every kernel loses what the saved mean's rounding
    costs, 2^-24 of the mean in units of the deviation, and no more."""
    offset = 1e4
    x, w, b, dy = _problem(rows, cols, F32, 3, offset)
    ref, tol = _reference(x, w, b, dy, 1e-5)
    y, mean, rstd = ops.layer_norm(x, w, b, stats=True)
    dx, dw, db = ops.layer_norm_backward(dy, x, w, mean, rstd)
    r = rstd.double().unsqueeze(1)
    slack = offset * 1.01 * 2.0 ** -24 * r  # of xhat
    a = (dy * w).double().abs()
    m = a.mean(1, keepdim=True)
    xh = ((x.double() - x.double().mean(1, keepdim=True)) * r).abs()
    # dx = rstd (a - mean(a) - xhat mean(a xhat)): xhat twice, the second under a mean
    grow = slack * (a * xh).mean(1, keepdim=True) + (xh + slack) * slack * m
    _check("dx", dx, ref["dx"], tol["dx"] + r * grow)
    _check("dw", dw, ref["dw"], tol["dw"] + (dy.double().abs() * slack).sum(0))
    _check("db", db, ref["db"], tol["db"])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,cols", [(80000, 256), (12001, 512), (20001, 300), (6000, 8192)])
def test_many_rows_a_block(cuda_device, rows, cols, dtype):
    """More than 32 rows in turn for a block: the rows' statistics are loaded
    again.  dweight and dbias are sums of `rows` terms in chains a block and trees
    over the blocks: with the chains' length against 96 roundings."""
    x, w, b, dy = _problem(rows, cols, dtype, rows)
    ref, tol = _reference(x, w, b, dy, 1e-5)
    y, mean, rstd = ops.layer_norm(x, w, b, stats=True)
    dx, dw, db = ops.layer_norm_backward(dy, x, w, mean, rstd)
    longer = max(1.0, rows / 148 / 96)  # rows of a block, at least one on each SM
    for k, got in (("y", y), ("dx", dx), ("dw", dw), ("db", db)):
        _check(k, got, ref[k], tol[k] * (longer if k in ("dw", "db") else 1.0))
