"""More GPU tests of the gated linear layer, with the checks and tolerances of
test_gated_gpu.py."""
from __future__ import annotations

import pytest
import torch

from moonxi_net_b200 import ops
from test_gated_gpu import _act, _halves, _problem, _run_and_check

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh"])
@pytest.mark.parametrize("M", [33, 95, 130, 289, 2059])
def test_warps_whose_lanes_part(cuda_device, M, act):
    """Rows that end inside a warp, under activations that branch on their
    values: what a warp does together comes after what its lanes do alone."""
    for F in (37, 264):
        _run_and_check(M, 128, F, BF16, False, act, True, seed=M + F)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_clusters_whose_lanes_part(cuda_device, dtype):
    """Few columns and a long K: eight blocks share a group of columns, and each
    finishes a few outputs with a few lanes of a warp."""
    for M in (1, 2, 4):
        for F in (1, 9, 40):
            _run_and_check(M, 4096, F, dtype, False, "gelu", True, seed=M + F)


@pytest.mark.parametrize("tw", [False, True])
@pytest.mark.parametrize("M,K,F", [(512, 1024, 2048), (40, 2048, 1000), (300, 4096, 72), (1000, 72, 301)])
def test_float32_tensor_products_keep_float32(cuda_device, M, K, F, tw):
    """The forward products and both gradients on the tensor cores, whole and with
    the K range in parts: each k-block's sum is truncated at most 24 times, the last
    few at full size, and rounded once: below 8 * 2^-24 of the result's norm, which
    sums of k-blocks of random sign keep; dpre is off by a few units in the last
    place more.  Held to 1e-6 of the norm; without the third bfloat16 copy of an
    operand it would be 2^-18, 4e-6."""
    x, w, b, dh = _problem(M, K, F, F32, tw, True, seed=M)
    kw = dict(act="silu", transpose_w=tw, precision="3xtf32")  # the tensor cores, whatever the shape
    h, pre = ops.gated_linear(x, w, b, save=True, **kw)
    dx, dw, db = ops.gated_linear_backward(dh, pre, x, w, **kw)
    X, W, D = x.double(), w.double().t() if tw else w.double(), dh.double()
    P = X @ W + b.double()
    a, da = _act("silu", P[:, :F])
    dp = torch.cat((D * P[:, F:] * da, D * a), 1)
    want = {"pre": P, "h": a * P[:, F:], "dx": dp @ W.t(), "dw": X.t() @ dp, "db": dp.sum(0)}
    got = {"pre": _halves(pre, F), "h": h, "dx": dx, "dw": dw.t() if tw else dw, "db": db}
    for k in want:
        off = float((got[k].double() - want[k]).norm() / want[k].norm())
        assert off < 1e-6, (k, off)


def test_long_and_thin_products(cuda_device):
    """42 million rows through weights that are not zero.  All values are small
    multiples of powers of two, so that every sum but the last few, where parts
    are joined, is exact: four roundings."""
    M, K, F = 42_000_001, 8, 8
    x = torch.full((M, K), 0.5, device="cuda")
    row = torch.tensor([1.0, 0.5, 0.25] * 3, device="cuda")[:K]
    col = torch.tensor([0.25, 0.5] * F, device="cuda")
    w = row[:, None] * col
    b = torch.ones(2 * F, device="cuda")
    h, pre = ops.gated_linear(x, w, b, act="relu", save=True)
    g = 0.5 * float(row.sum()) * col.double() + 1  # of every row
    a, u = g[:F], g[F:]
    assert (h.double() == a * u).all()
    dx, dw, db = ops.gated_linear_backward(h.fill_(0.25), pre, x, w, act="relu")
    dp = torch.cat((0.25 * u, 0.25 * a))
    assert (dx.double() == w.double() @ dp).all()
    tol = 4 * 2.0 ** -24
    assert ((dw.double() / (0.5 * M * dp) - 1).abs() <= tol).all()
    assert ((db.double() / (M * dp) - 1).abs() <= 4 * tol).all()
