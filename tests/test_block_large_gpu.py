"""GPU tests of tensors with more than 2^31 elements: what lies beyond is
computed as the same rows (or values) are in a small call."""
from __future__ import annotations

import pytest
import torch

from moonxi_net_b200 import nn, ops

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def _far_rows(rows):
    """The first rows, those around 2^31 and 2^32 bytes and elements, the last."""
    return torch.unique(torch.cat([torch.arange(3), torch.arange(rows - 3, rows)]
                                  + [torch.arange(k - 2, k + 2) for k in (rows // 4, rows // 2)]))


@pytest.mark.parametrize("cols", [8192, 8191])
def test_layer_norm(cuda_device, cols):
    rows = 2 ** 31 // cols + 200
    g = torch.Generator("cuda").manual_seed(1)
    x = torch.empty(rows, cols, device="cuda", dtype=BF16).normal_(generator=g)
    w, b = (torch.randn(cols, device="cuda", generator=g) for _ in range(2))
    y, mean, rstd = ops.layer_norm(x, w, b, stats=True)
    at = _far_rows(rows).cuda()
    xs = x[at]
    ys, ms, rs = ops.layer_norm(xs, w, b, stats=True)
    assert torch.equal(y[at], ys) and torch.equal(mean[at], ms) and torch.equal(rstd[at], rs)
    # y as the gradient; these few rows alone have one that is not zero, so that
    # the sums over all rows are theirs
    dy = torch.zeros_like(x)
    dy[at] = ys
    del y
    dx, dw, db = ops.layer_norm_backward(dy, x, w, mean, rstd)
    ref, dws, dbs = ops.layer_norm_backward(ys, xs, w, ms, rs)
    # two kernels for so different numbers of rows: a few roundings of float32
    # of sums over a row apart, and one of bfloat16
    assert (dx[at].double() - ref.double()).abs().max() <= 2.0 ** -7 * ref.double().abs().max()
    for got, want in ((dw, dws), (db, dbs)):
        assert ((got - want).abs() <= 2.0 ** -18 * want.abs().max()).all()


@pytest.mark.parametrize("F", [16, 13])
def test_gated_linear(cuda_device, F):
    K = 8192
    M = 2 ** 31 // K + 300
    g = torch.Generator("cuda").manual_seed(2)
    x = torch.empty(M, K, device="cuda", dtype=BF16).normal_(generator=g)
    w = (torch.randn(K, 2 * F, device="cuda", generator=g) / K ** 0.5).to(BF16)
    h, pre = ops.gated_linear(x, w, save=True)
    at = _far_rows(M).cuda()
    P = x[at].double() @ w.double()
    got = torch.cat((pre[at][:, :F], pre[at][:, pre.shape[1] // 2:][:, :F]), 1).double()
    E = (K / 16 + 40) * 2.0 ** -23 * (x[at].double().abs() @ w.double().abs())
    assert ((got - P).abs() <= E).all()
    dh = torch.zeros_like(h)
    dh[at] = 1.0
    dx, dw, db = ops.gated_linear_backward(dh, pre, x, w)
    gp, up = P[:, :F], P[:, F:]
    s = torch.sigmoid(gp)
    dp = torch.cat((up * s * (1 + gp * (1 - s)), gp * s), 1)
    # dpre and the result are rounded to bfloat16, 2^-8 each, and g and u are off by E
    for got, want, terms in ((dx[at], dp @ w.double().t(), dp.abs() @ w.double().abs().t()),
                             (dw, x[at].double().t() @ dp, x[at].double().abs().t() @ dp.abs()),
                             (db, dp.sum(0), dp.abs().sum(0))):
        assert ((got.double() - want).abs() <= 2.0 ** -8 * (want.abs() + terms) * 1.01 + 1e-3 * E.max()).all()
    rest = torch.ones(M, dtype=torch.bool, device="cuda")
    rest[at] = False
    assert not dx[rest].any()


@pytest.mark.parametrize("kind", ["f32", "codes"])
def test_adamw(cuda_device, kind):
    n = 2 ** 31 + 5000 if kind == "codes" else 2 ** 30 + 5000
    kw = dict(state_bits=8 if kind == "codes" else 32, betas=(0.9, 0.95))
    p = torch.zeros(n, device="cuda")
    g = torch.zeros(n, device="cuda", dtype=BF16)
    g[-5000:] = torch.randn(5000, device="cuda", generator=torch.Generator("cuda").manual_seed(3)).to(BF16)
    start = n - n % 256 - 256 * 30  # on a block of 256 of its own
    opt = nn.AdamW([p], **kw)
    ref = nn.AdamW([p[start:].clone()], **kw)
    for _ in range(2):
        opt.step([g])
        ref.step([g[start:].clone()])
    assert torch.equal(p[start:], ref.params[0]) and p[start:].any()
    assert not p[:n - 5000].any()
    m, want = opt.state[0][0][start:], ref.state[0][0]
    assert torch.equal(m, want)
