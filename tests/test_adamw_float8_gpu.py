"""GPU tests of nn.AdamW on 8-bit floating-point moments (float8_e4m3fn values,
each times a power of two that its 256 values share), against the same step in
elementary float32 operations, which it gives bit for bit: every operation is
rounded by itself, and which of two neighbours a value becomes depends on it."""
from __future__ import annotations

import math

import pytest
import torch

from moonxi_net_b200 import _lib, nn, ops

pytestmark = pytest.mark.gpu
F32, BF16, F8 = torch.float32, torch.bfloat16, torch.float8_e4m3fn
HYPER = dict(lr=1e-3, betas=(0.9, 0.9), eps=1e-8, weight_decay=0.1)
SIZES = [1, 7, 8, 255, 256, 257, 2048, 5003, 70001]


def _encode(x):
    n = x.numel()
    x = torch.nn.functional.pad(x, (0, -n % 256)).view(-1, 256)
    top = x.abs().amax(1, keepdim=True).clamp(min=2.0 ** -119)
    scale = (top.view(torch.int32) & 0x7F800000).view(F32) * 2.0 ** -7
    y = x / scale
    least = torch.full_like(y, 2.0 ** -9)
    y = torch.where((y != 0) & (y.abs() < 2.0 ** -9), torch.copysign(least, y), y)
    return y.to(F8).view(-1)[:n], scale.view(-1)


def _decode(q, scale):
    return q.float() * scale.repeat_interleave(256)[:q.numel()]


def _plain(p, g, state, t, lr, betas, eps, weight_decay):
    """The step in float32, an operation at a time; the new p and state."""
    (b1, b2), g = betas, g.float()
    m = _decode(*state[:2]) * b1 + g * (1 - b1)
    v = _decode(*state[2:]).square() * b2 + (g * g) * (1 - b2)
    root = v.sqrt()
    denom = root * (1 / math.sqrt(1 - b2 ** t)) + eps
    p = p * (1 - lr * weight_decay) - (m * (lr / (1 - b1 ** t))) / denom
    return p, (*_encode(m), *_encode(root))


def _zero_state(n):
    return (torch.zeros(n, device="cuda", dtype=F8), torch.zeros(-(-n // 256), device="cuda"),
            torch.zeros(n, device="cuda", dtype=F8), torch.zeros(-(-n // 256), device="cuda"))


def _randn(n, seed, scale=1.0, dtype=F32):
    g = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn(n, device="cuda", generator=g) * scale).to(dtype)


def _same(a, b):
    """Equal bits; NaNs are alike."""
    a, b = a.float(), b.float()
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_steps_are_the_plain_ones(cuda_device, dtype):
    ps = [_randn(n, i, 0.1) for i, n in enumerate(SIZES)]
    copies = [torch.zeros(n, device="cuda", dtype=BF16) for n in SIZES]
    opt = nn.AdamW(ps, state_bits=8, state=[_zero_state(n) for n in SIZES], copies=copies, **HYPER)
    want = [(p.clone(), _zero_state(p.numel())) for p in ps]
    for t in range(1, 6):
        # values of very different size, and some without a gradient
        gs = [(_randn(n, 100 * t + i, 0.01) * torch.exp(3 * _randn(n, 7 * i))
               * (_randn(n, 9 * i) > -1)).to(dtype) for i, n in enumerate(SIZES)]
        opt.step(gs)
        want = [_plain(p, g, s, t, **HYPER) for (p, s), g in zip(want, gs)]
        for p, c, s, (wp, ws) in zip(opt.params, copies, opt.state, want):
            assert torch.equal(p, wp) and torch.equal(c, wp.to(BF16))
            assert all(_same(x, y) for x, y in zip(s, ws))


def test_unaligned_and_resumed(cuda_device):
    n = 1000
    g = _randn(n, 1, 0.01)
    a = nn.AdamW([_randn(n, 2)], state_bits=8, state=[_zero_state(n)], **HYPER)

    def off(t):
        return torch.empty(t.numel() + 3, device="cuda", dtype=t.dtype)[3:].copy_(t)
    s = tuple(off(x) for x in _zero_state(n))
    b = nn.AdamW([off(_randn(n, 2))], state_bits=8, state=[s], **HYPER)
    for _ in range(2):
        a.step([g])
        b.step([off(g)])
    b = nn.AdamW(b.params, state_bits=8, state=b.state, step_count=b.step_count, **HYPER)
    a.step([g])
    b.step([g])
    assert torch.equal(a.params[0], b.params[0])
    assert all(_same(x, y) for x, y in zip(a.state[0], b.state[0]))


def test_tiny_zero_and_not_finite(cuda_device):
    n = 256 * 6
    p, g = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    g[256:512] = _randn(256, 1) * 2.0 ** -117
    g[512:768] = _randn(256, 1) * 2.0 ** -100
    g[768] = float("inf")
    g[1024] = float("nan")
    g[1025:1280] = 1.0
    g[1280:] = _randn(256, 1) * 1e18
    opt = nn.AdamW([p], state_bits=8, state=[_zero_state(n)], **HYPER)
    want = (p.clone(), _zero_state(n))
    for t in (1, 2, 3):
        opt.step([g])
        want = _plain(want[0], g, want[1], t, **HYPER)
        assert _same(p, want[0])
        assert all(_same(x, y) for x, y in zip(opt.state[0], want[1]))
    assert (p[:256] == 0).all() and (opt.state[0][0][:256].float() == 0).all()


def test_refusals(cuda_device):
    p = torch.ones(300, device="cuda")
    s = _zero_state(300)
    codes = nn.AdamW([p.clone()], state_bits=8).state[0]
    with pytest.raises(TypeError):  # the two kinds of 8-bit state do not mix
        nn.AdamW([p], state_bits=8, state=[(s[0], s[1], codes[2], codes[3])], **HYPER)
    with pytest.raises(TypeError):
        nn.AdamW([p, p.clone()], state_bits=8, state=[s, codes], **HYPER)
    with pytest.raises(TypeError):
        nn.AdamW([p], state_bits=8, state=[(s[0].view(torch.uint8).view(torch.float8_e5m2), *s[1:])], **HYPER)
    with pytest.raises(TypeError):
        nn.AdamW([p], state=[(s[0], s[2])], **HYPER)
    with pytest.raises(ValueError):
        nn.AdamW([p], state_bits=8, state=[(s[0], s[1][:1], s[2], s[3])], **HYPER)
    L, h = _lib.lib(), ops.context(0)
    t = (_lib.AdamWTensor * 1)()
    for bits in (32 | _lib.ADAMW_E4M3, 8 | 0x1000, _lib.ADAMW_E4M3):
        assert L.mx_adamw_step(h, t, 1, bits, 1e-3, 0.9, 0.9, 1e-8, 1, None, 0.0, None, None, 0,
                               None) == _lib.MX_ERR_INVALID
