"""Layer norm, the gated linear layer and AdamW as they are used together: a
pre-norm gated feed-forward block between the framework's own products and its
cross-entropy, trained for some steps.

    y = x + gated(norm(x)) w_out,  logits = y w_head,  loss = CE(logits, labels)

Tolerances.  float32: ten operations whose sums run over at most 300 terms: each
is off by less than 300 * 2^-24 of its terms' sum, which for terms of random sign
is at most sqrt(300) times the result: 10 * 300 * 2^-24 * 17.3 = 3.1e-3 of a
gradient's norm.  bfloat16 (x, the gated layer and its gradients): seven values on
the longest way are rounded by 2^-8 each, 2.7e-2, on top of that.
"""
from __future__ import annotations

import pytest
import torch

from moonxi_net_b200 import nn, ops

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
M, D, F, C = 144, 96, 168, 40


class Block:
    """The block's parameters (float32, and bfloat16 copies of the gated
    layer's when dtype is bfloat16), its step and its optimizer."""

    def __init__(self, dtype, bits, device_step=False, max_grad_norm=1.0):
        g = torch.Generator("cuda").manual_seed(0)

        def randn(*s, scale):
            return torch.randn(*s, device="cuda", generator=g) * scale
        self.dtype = dtype
        self.p = {"gain": 1 + randn(D, scale=0.1), "shift": randn(D, scale=0.1),
                  "w_in": randn(D, 2 * F, scale=D ** -0.5), "b_in": randn(2 * F, scale=0.1),
                  "w_out": randn(F, D, scale=F ** -0.5), "w_head": randn(D, C, scale=D ** -0.5)}
        low = ("w_in", "b_in") if dtype is BF16 else ()
        self.low = {k: self.p[k].to(BF16) for k in low}
        names = list(self.p)
        self.opt = nn.AdamW([self.p[k] for k in names], lr=1e-2, state_bits=bits,
                            copies=[self.low.get(k) for k in names],
                            weight_decay=[0.1 if self.p[k].dim() == 2 else 0.0 for k in names],
                            max_grad_norm=max_grad_norm, device_step=device_step)

    def gradients(self, x, labels):
        p, low, t = self.p, self.low, self.dtype
        xn, mean, rstd = ops.layer_norm(x, p["gain"], p["shift"], stats=True)
        w, b = low.get("w_in", p["w_in"]), low.get("b_in", p["b_in"])
        h, pre = ops.gated_linear(xn, w, b, act="silu", save=True)
        hf, xf = h.float(), x.float()
        y = xf.clone()
        ops.matmul(hf, p["w_out"], M, F, D, beta=1.0, out=y)
        logits = ops.matmul(y, p["w_head"], M, D, C)
        loss, dlog = ops.softmax_ce_labels(logits, labels)
        dy = ops.matmul(dlog, p["w_head"], M, C, D, tb=True)
        g = {"w_head": ops.matmul(y, dlog, D, M, C, ta=True),
             "w_out": ops.matmul(hf, dy, F, M, D, ta=True)}
        dh = ops.matmul(dy, p["w_out"], M, D, F, tb=True)
        dxn, g["w_in"], g["b_in"] = ops.gated_linear_backward(dh.to(t), pre, xn, w)
        dx, g["gain"], g["shift"] = ops.layer_norm_backward(dxn, x, p["gain"], mean, rstd)
        return loss, g, dy + dx.float()

    def step(self, x, labels):
        loss, g, _ = self.gradients(x, labels)
        self.opt.step([g[k] for k in self.p])
        return loss


def _batch(dtype, seed=1):
    g = torch.Generator("cuda").manual_seed(seed)
    x = torch.randn(M, D, device="cuda", generator=g).to(dtype)
    return x, torch.randint(0, C, (M,), device="cuda", generator=g).float()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gradients_of_the_whole_block(cuda_device, dtype):
    blk = Block(dtype, 32)
    x, labels = _batch(dtype)
    loss, got, dx = blk.gradients(x, labels)
    leaves = {k: v.double().requires_grad_() for k, v in {**blk.p, **blk.low}.items()}
    xd = x.double().requires_grad_()
    mean = xd.mean(1, keepdim=True)
    xn = (xd - mean) / (((xd - mean) ** 2).mean(1, keepdim=True) + 1e-5).sqrt()
    xn = xn * leaves["gain"] + leaves["shift"]
    pre = xn @ leaves["w_in"] + leaves["b_in"]
    h = pre[:, :F] * torch.sigmoid(pre[:, :F]) * pre[:, F:]
    logits = (xd + h @ leaves["w_out"]) @ leaves["w_head"]
    want = -torch.log_softmax(logits, 1).gather(1, labels.long()[:, None]).mean()
    grads = torch.autograd.grad(want, [*leaves.values(), xd])
    tol = 3.1e-3 + (7 * 2.0 ** -8 if dtype is BF16 else 0.0)
    want = want.detach()
    assert abs(float(loss) - float(want)) <= tol * abs(float(want))
    for k, w in zip([*leaves, "x"], grads):
        g = dx if k == "x" else got[k]
        assert float((g.double() - w).norm()) <= tol * float(w.norm()), k


@pytest.mark.parametrize("dtype,bits", [(F32, 32), (F32, 8), (BF16, 32), (BF16, 8)])
def test_steps_run_and_a_captured_step_replays_them(cuda_device, dtype, bits):
    """Eager steps and replays of one captured step give the same bits."""
    a, b = Block(dtype, bits), Block(dtype, bits, device_step=True)
    x, labels = _batch(dtype)
    b.gradients(x, labels)  # the products' workspace, before the capture
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss_b = b.step(x, labels)
    for i in range(6):
        xi, li = _batch(dtype, 10 + i)
        x.copy_(xi)
        labels.copy_(li)
        graph.replay()
        loss_a = a.step(xi, li)
        assert torch.equal(loss_a, loss_b) and loss_a.isfinite().all()
    for k in a.p:
        assert torch.equal(a.p[k], b.p[k]), k
    for k in a.low:
        assert torch.equal(a.low[k], b.low[k]) and torch.equal(a.low[k], a.p[k].to(BF16)), k
    assert a.opt.step_count == 6 and int(b.opt.step_dev) == 6
    assert ops.status() == (0, 0)
