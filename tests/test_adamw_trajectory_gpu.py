"""GPU tests of nn.AdamW's 8-bit moments over many steps, against a run in 64 bits
that never sees the stored states.

Gradients of eight sizes stand in each block of 256 values, some of which shrink
by ten and some of which grow by ten while the block's largest stays, so that
their codes have to move against it by changes far below a code a step.

Tolerances.  Rounding without bias leaves a value's moment right on the average
over the N = 16384 values of a size.  One step's rounding has a deviation of at
most half of a code's step: relatively 2 / k of v at code k (of 255; v goes with
k^4), 1 / k of m (of 127; m goes with k^2); float8 values have steps of at most
1/8, of v twice that: 1/8 and 1/16.  Roundings die out with the moment's memory: the
deviations of 1 / (1 - beta^2) steps add up as a root.  Six deviations of the mean
of N are allowed, and 1 % for what the steps' own moments are off by.
"""
from __future__ import annotations

import math

import pytest
import torch

from moonxi_net_b200 import nn

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn
# each size's gradient at first and later, against the largest of the block
SIZES = [(1.0, 1.0), (0.5, 0.05), (0.05, 0.5), (0.2, 0.02), (0.02, 0.2), (0.1, 0.01), (0.01, 0.1), (0.3, 0.3)]
BLOCKS = 512
N = BLOCKS * 32


def _decode(state):
    mq, ms, vq, vs = state
    ms, vs = (x.double().repeat_interleave(256) for x in (ms, vs))
    if mq.dtype is F8:
        return mq.double() * ms, (vq.double() * vs) ** 2
    m, v = mq.double(), vq.double()
    return m.sign() * (m / 127) ** 2 * ms, ((v / 255) ** 2 * vs) ** 2


def _state(kind, n):
    if kind == "codes":
        return None
    return [(torch.zeros(n, device="cuda", dtype=F8), torch.zeros(n // 256, device="cuda"),
             torch.zeros(n, device="cuda", dtype=F8), torch.zeros(n // 256, device="cuda"))]


def _run(kind, betas, steps, change, **kw):
    """The optimizer's moments and those of 64 bits, a row for each size."""
    n = BLOCKS * 256
    gen = torch.Generator("cuda").manual_seed(1)
    p = torch.zeros(n, device="cuda")
    opt = nn.AdamW([p], lr=1e-3, betas=betas, weight_decay=0.0, state_bits=8, state=_state(kind, n), **kw)
    m, v = (torch.zeros(n, device="cuda", dtype=torch.double) for _ in range(2))
    size = [torch.tensor([s[i] for s in SIZES], device="cuda").repeat(n // 8) for i in (0, 1)]
    for t in range(steps):
        g = size[t >= change] * (1 + 0.3 * torch.randn(n, device="cuda", generator=gen))
        opt.step([g])
        m.lerp_(g.double(), 1 - betas[0])
        v.lerp_(g.double() ** 2, 1 - betas[1])
    rows = [x.view(-1, 8).t() for x in (*_decode(opt.state[0]), m, v)]
    return rows


@pytest.mark.parametrize("kind", ["codes", "float8"])
@pytest.mark.parametrize("betas", [(0.9, 0.999), (0.9, 0.99), (0.95, 0.95)])
def test_moments_follow(cuda_device, kind, betas):
    """The class's default betas, and others near one."""
    got_m, got_v, m, v = _run(kind, betas, 1200, 200)
    top_m, top_v = m.abs().mean(1).max(), v.mean(1).max()
    for i in range(8):
        if kind == "codes":
            dev_m = 1 / (127 * float(m[i].mean() / top_m) ** 0.5)
            dev_v = 2 / (255 * float(v[i].mean() / top_v) ** 0.25)
        else:
            dev_m, dev_v = 1 / 16, 1 / 8
        for name, got, want, dev, beta in (("m", got_m, m, dev_m, betas[0]), ("v", got_v, v, dev_v, betas[1])):
            tol = 0.01 + 6 * dev / math.sqrt((1 - beta * beta) * N)
            ratio = float(got[i].mean() / want[i].mean())
            assert abs(ratio - 1) <= tol, (name, SIZES[i], ratio, tol)


@pytest.mark.parametrize("kind", ["codes", "float8"])
def test_dead_values(cuda_device, kind):
    """Where gradients stop, first moments reach zero, although others of the
    block go on, and the values then stay; second moments stay above zero."""
    p = torch.zeros(256, device="cuda")
    opt = nn.AdamW([p], state_bits=8, lr=0.01, state=_state(kind, 256), weight_decay=0.0)
    g = torch.full((256,), 1.0, device="cuda")
    opt.step([g])
    g[:128] = 0
    # m halves in 7 steps; from the smallest value on each step keeps it with a
    # chance of 0.9, so that after 500 more none of 128 is left (128 * 0.9^500)
    for _ in range(700):
        opt.step([g])
    m, v = _decode(opt.state[0])
    assert (m[:128] == 0).all() and (v[:128] > 0).all() and (m[128:] > 0).all()
    before = p[:128].clone()
    opt.step([g])
    assert torch.equal(p[:128], before)


@pytest.mark.parametrize("kind", ["codes", "float8"])
def test_rounding_repeats(cuda_device, kind):
    """How a value is rounded depends on the step's number and its place alone:
    resumed, captured and repeated runs give the same bits."""
    n = 5 * 256
    gen = torch.Generator("cuda").manual_seed(3)
    gs = [torch.randn(n, device="cuda", generator=gen) for _ in range(6)]

    def make(p, state, **kw):
        return nn.AdamW([p], state_bits=8, state=state, **kw)
    a, b, c = (make(torch.ones(n, device="cuda"), _state(kind, n), **kw)
               for kw in ({}, {}, {"device_step": True}))
    held = torch.empty(n, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.step([held])
    for t, g in enumerate(gs):
        if t == 3:
            b = make(b.params[0], b.state, step_count=b.step_count)
        a.step([g])
        b.step([g])
        held.copy_(g)
        graph.replay()
    for o in (b, c):
        assert torch.equal(a.params[0], o.params[0])
        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a.state[0], o.state[0]))
    again = make(torch.ones(n, device="cuda"), _state(kind, n))
    for g in gs[:5] + [gs[5]]:
        again.step([g])
    assert torch.equal(again.params[0], a.params[0])


def test_rounding_is_an_argument(cuda_device):
    """Nearest codes where beta1 is at most 0.9 and beta2 at most 0.97, unless the
    caller says; what is held in 32 bits is not rounded."""
    g = torch.linspace(-1, 1, 2560, device="cuda")

    def codes(**kw):
        opt = nn.AdamW([torch.zeros(2560, device="cuda")], state_bits=8, **kw)
        for _ in range(3):
            opt.step([g])
        return opt.state[0][2]
    near = codes(betas=(0.9, 0.97))
    assert torch.equal(near, codes(betas=(0.9, 0.97), rounding="nearest"))
    assert not torch.equal(near, codes(betas=(0.9, 0.97), rounding="dither"))
    far = codes(betas=(0.9, 0.98))
    assert torch.equal(far, codes(betas=(0.9, 0.98), rounding="dither"))
    assert not torch.equal(far, codes(betas=(0.9, 0.98), rounding="nearest"))
    assert (near.int() - codes(betas=(0.9, 0.97), rounding="dither").int()).abs().max() <= 3
    with pytest.raises(ValueError, match="rounding"):
        nn.AdamW([g], state_bits=8, rounding="up")
    with pytest.raises(ValueError, match="rounding"):
        nn.AdamW([g], rounding="dither")
    with pytest.warns(UserWarning, match="never fall"):
        nn.AdamW([g], state_bits=8, betas=(0.9, 0.95), state=_state("float8", 2560))


@pytest.mark.parametrize("kind", ["codes", "float8"])
def test_zero_and_not_finite_values(cuda_device, kind):
    """Rounded up or down, zero stays zero, in blocks of zeros and in others; what
    is not finite reaches its block and no further."""
    n = 256 * 5
    g = torch.zeros(n, device="cuda")
    g[256:512:2] = torch.randn(128, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    g[512:768] = 2.0 ** -100
    p = torch.zeros(n, device="cuda")
    opt = nn.AdamW([p], state_bits=8, state=_state(kind, n), weight_decay=0.0)
    for _ in range(5):
        opt.step([g])
    m, v = _decode(opt.state[0])
    zero = g == 0
    assert (m[zero] == 0).all() and (v[zero] == 0).all() and (p[zero] == 0).all()
    assert (m[256:512:2] != 0).all() and (v[256:512:2] > 0).all()
    before = [x.clone() for x in opt.state[0]]
    for bad in (math.inf, -math.inf, math.nan):
        state = [tuple(x.clone() for x in before)]
        other = nn.AdamW([p.clone()], state_bits=8, state=state, step_count=5, weight_decay=0.0)
        good = nn.AdamW([p.clone()], state_bits=8, state=[tuple(x.clone() for x in before)], step_count=5,
                        weight_decay=0.0)
        g2 = g.clone()
        g2[300] = bad
        other.step([g2])
        good.step([g])
        keep = torch.arange(n, device="cuda") // 256 != 1
        (ma, va), (mb, vb) = _decode(other.state[0]), _decode(good.state[0])
        assert torch.equal(ma[keep], mb[keep]) and torch.equal(va[keep], vb[keep])
        ok = torch.arange(n, device="cuda") != 300
        assert torch.equal(other.params[0][ok], good.params[0][ok]) and other.params[0][300].isnan()
        assert not ma[300].isfinite() and not va[300].isfinite()
