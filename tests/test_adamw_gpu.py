"""GPU tests of nn.AdamW (mx_adamw_step) against the step in 64 bits.

Tolerances, with u = 2^-24.  m is a sum of two terms, each the product of a
rounded constant: 3 u of |b1 m| + |(1 - b1) g|, not of m itself, since the terms
may cancel.  v's terms cannot: 4 u v.  In the update lr/c1 m / (sqrt(v)/c2 + eps)
the numerator adds a constant and a product (2 u) to m's own error, which
counts as lr/c1 / denominator of it; the root of v is off by 2 u + u, the
denominator by a constant, a product and a sum more (6 u), the quotient by u: 9 u
|update| and m's share.  p adds the decay's constant and product and the
result's rounding: 2 u |p| + u |new p|.  With 8-bit moments the root and the
reciprocal are approximate (2 u and 2 u): 16 u.  An 8-bit code is the nearest one in the root: off by at
most half a step, and 2^-10 of a step for the root's own last bits; small codes
of m are floor(root + 1/64) instead.
"""
from __future__ import annotations

import pytest
import torch

from moonxi_net_b200 import _lib, nn, ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16
HYPER = dict(lr=3e-3, betas=(0.9, 0.97), eps=1e-8, weight_decay=0.05)
# one value, below a vector, a block of 256 and its neighbours, a chunk and more
SIZES = [1, 5, 8, 255, 256, 257, 2048, 2049, 5000, 70001]


def _randn(n, seed, scale=1.0, dtype=F32):
    g = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn(n, device="cuda", generator=g) * scale).to(dtype)


def _tensors(sizes, grad_types, seed=0):
    ps = [_randn(n, seed + i, 0.1) for i, n in enumerate(sizes)]
    gs = [_randn(n, seed + 100 + i, 0.01, grad_types[i % len(grad_types)]) for i, n in enumerate(sizes)]
    return ps, gs


def _decode(codes, scale):
    top = scale.double().repeat_interleave(256)[:codes.numel()]
    c = codes.double()
    if codes.dtype == torch.int8:
        return c.sign() * (c / 127) ** 2 * top
    return ((c / 255) ** 2 * top) ** 2


def _moments(state):
    if len(state) == 2:
        return state[0].double(), state[1].double()
    return _decode(state[0], state[1]), _decode(state[2], state[3])


def _step64(p, g, m, v, t, lr, betas, eps, weight_decay, clip=1.0):
    b1, b2 = betas
    g = g.double() * clip
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    upd = lr / (1 - b1 ** t) * m / (v.sqrt() / (1 - b2 ** t) ** 0.5 + eps)
    return p.double() * (1 - lr * weight_decay) - upd, m, v, upd


def _check_step(opt, before, grads, t, clip=1.0, decay=None):
    """One step, already taken, against 64 bits from the state before it."""
    slack = 4 * U if clip != 1.0 else 0.0  # the clip factor's roundings
    for i, (p, (p0, m0, v0), g) in enumerate(zip(opt.params, before, grads)):
        h = dict(HYPER, weight_decay=HYPER["weight_decay"] if decay is None else decay[i])
        want, m, v, upd = _step64(p0, g, m0, v0, t, clip=clip, **h)
        k = 16 if opt.state_bits == 8 else 9
        gc = g.double().abs() * clip
        em = 3 * U * (0.9 * m0.abs() + 0.1 * gc) + slack * 0.1 * gc
        denom = v.sqrt() / (1 - 0.97 ** t) ** 0.5 + HYPER["eps"]
        lim = U * (2 * p0.double().abs() + want.abs()) + (k * U + 4 * slack) * upd.abs() \
            + HYPER["lr"] / (1 - 0.9 ** t) * em / denom
        assert ((p.double() - want).abs() <= lim).all(), i
        ev = 4 * U * v + 2 * slack * v
        if opt.state_bits == 32:
            m1, v1 = _moments(opt.state[i])
            assert ((m1 - m).abs() <= em).all() and ((v1 - v).abs() <= ev).all(), i
            continue
        mq, ms, vq, vs = opt.state[i]
        for codes, scale, x, ex, most in ((mq, ms, m, em, 127), (vq, vs, v.sqrt(), ev / (2 * v.sqrt() + 1e-30), 255)):
            n = x.numel()
            pad = torch.nn.functional.pad(x.abs(), (0, -n % 256)).view(-1, 256)
            top = pad.amax(1).clamp_min(2.0 ** -120)
            assert ((scale.double() - top).abs() <= 16 * U * top).all()
            root = (x.abs() / top.repeat_interleave(256)[:n]).sqrt() * most
            near = torch.sqrt((x.abs() + ex) / top.repeat_interleave(256)[:n]) * most - root
            off = (codes.double().abs() - root).abs()
            ok = off <= 0.5 + 2.0 ** -10 + near
            if most == 255:  # what is above zero stays above zero
                ok |= (codes == 1) & (root < 1)
                assert ((codes > 0) == (x > 0)).all()
            else:
                low = root < 0.5 / (1 - 0.9 ** 0.5) + 1
                c, slack8 = codes.double().abs(), 2.0 ** -10 + near
                down = (c <= root + 1 / 64 + slack8) & (c > root + 1 / 64 - 1 - slack8)
                border = (root - (0.5 / (1 - 0.9 ** 0.5) + 1)).abs() <= slack8
                ok = torch.where(low, down | (border & ok), ok | (border & down))
                assert ((codes == 0) | (codes.double().sign() == x.sign())).all()
            assert ok.all(), (i, float(off.max()))


def _before(opt):
    return [(p.clone(), *(x.clone() for x in _moments(s))) for p, s in zip(opt.params, opt.state)]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("grad_types", [[F32], [BF16], [F32, BF16]])
def test_steps_against_64_bits(cuda_device, bits, grad_types):
    ps, _ = _tensors(SIZES, grad_types)
    copies = [torch.zeros(n, device="cuda", dtype=BF16) if i % 2 else None for i, n in enumerate(SIZES)]
    opt = nn.AdamW(ps, state_bits=bits, copies=copies, **HYPER)
    for t in range(1, 4):
        grads = _tensors(SIZES, grad_types, seed=10 * t)[1]
        before = _before(opt)
        opt.step(grads)
        _check_step(opt, before, grads, t)
    for p, c in zip(ps, copies):
        assert c is None or torch.equal(c, p.to(BF16))


@pytest.mark.parametrize("bits", [32, 8])
def test_clipping_by_the_global_norm(cuda_device, bits):
    decay = [0.0 if i % 2 else 0.1 for i in range(len(SIZES))]
    ps, gs = _tensors(SIZES, [F32, BF16])
    h = {k: v for k, v in HYPER.items() if k != "weight_decay"}
    opt = nn.AdamW(ps, state_bits=bits, weight_decay=decay, max_grad_norm=0.5, **h)
    norm = torch.stack([g.double().norm() for g in gs]).norm()
    assert float(norm) > 1.0
    before = _before(opt)
    opt.step(gs)
    # a chain of at most a block's chunks, then trees: 64 * 2^-24
    assert abs(float(opt.norm) - float(norm)) <= 64 * U * float(norm)
    _check_step(opt, before, gs, 1, clip=float(0.5 / opt.norm.double()), decay=decay)
    small = [(g.float() * 1e-3).to(g.dtype) for g in gs]  # below the limit: not clipped
    before = _before(opt)
    opt.step(small)
    _check_step(opt, before, small, 2, decay=decay)


@pytest.mark.parametrize("bits", [32, 8])
def test_unaligned_tensors_and_their_neighbours(cuda_device, bits):
    """Tensors packed one after the other, off 16 bytes; what lies between stays."""
    sizes = [3, 300, 1, 1000]
    gap = 5
    total = sum(sizes) + gap * (len(sizes) + 1)

    def packed(dtype, fill=0):
        buf = torch.full((total,), 9, device="cuda", dtype=dtype)
        views, at = [], gap
        for n in sizes:
            buf[at:at + n] = fill
            views.append(buf[at:at + n])
            at += n + gap
        return buf, views
    ps_ref, gs = _tensors(sizes, [F32, BF16])
    pb, ps = packed(F32)
    cb, cs = packed(BF16)
    for p, r in zip(ps, ps_ref):
        p.copy_(r)
    bufs = [pb, cb]
    if bits == 32:
        (mb, ms), (vb, vs) = packed(F32), packed(F32)
        state = list(zip(ms, vs))
    else:
        (mb, ms), (vb, vs) = packed(torch.int8), packed(torch.uint8)
        scales = [[torch.zeros(-(-n // 256), device="cuda") for n in sizes] for _ in range(2)]
        state = list(zip(ms, scales[0], vs, scales[1]))
    bufs += [mb, vb]
    opt = nn.AdamW(ps, state_bits=bits, copies=cs, state=state, **HYPER)
    ref = nn.AdamW([p.clone() for p in ps_ref], state_bits=bits, **HYPER)
    for _ in range(3):
        opt.step(gs)
        ref.step(gs)
    for a, b in zip(opt.params, ref.params):
        assert torch.equal(a, b)
    for sa, sb in zip(opt.state, ref.state):
        assert all(torch.equal(x, y) for x, y in zip(sa, sb))
    at = 0
    for n in sizes + [0]:
        for buf in bufs:
            assert (buf[at:at + gap] == 9).all()
        at += gap + n


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors(cuda_device, bits):
    """More tensors than one launch holds, empty ones among them."""
    sizes = [(i * 37) % 300 for i in range(700)]
    ps, gs = _tensors(sizes, [F32, BF16])
    opt = nn.AdamW(ps, state_bits=bits, max_grad_norm=1e-3, **HYPER)
    before = _before(opt)
    launches = _lib.lib().mx_kernel_launch_count()
    opt.step(gs)
    assert _lib.lib().mx_kernel_launch_count() - launches == 2 * 3 + 1
    norm = torch.cat([g.double() for g in gs]).norm()
    assert abs(float(opt.norm) - float(norm)) <= 64 * U * float(norm)
    _check_step(opt, before, gs, 1, clip=float(1e-3 / opt.norm.double()))


@pytest.mark.parametrize("bits", [32, 8])
def test_resumed_run_goes_on(cuda_device, bits):
    ps, _ = _tensors([700, 33], [F32])
    a = nn.AdamW([p.clone() for p in ps], state_bits=bits, **HYPER)
    for t in range(2):
        a.step(_tensors([700, 33], [F32], 7 + t)[1])
    b = nn.AdamW([p.clone() for p in a.params], state_bits=bits,
                 state=[tuple(x.clone() for x in s) for s in a.state], step_count=a.step_count, **HYPER)
    for t in range(2):
        gs = _tensors([700, 33], [F32], 50 + t)[1]
        a.step(gs)
        b.step(gs)
    assert all(torch.equal(x, y) for x, y in zip(a.params, b.params))
    assert a.step_count == b.step_count == 4


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step_counts_its_replays(cuda_device, bits):
    ps, gs = _tensors([1000, 257], [F32])
    eager = nn.AdamW([p.clone() for p in ps], state_bits=bits, max_grad_norm=0.1, **HYPER)
    dev = nn.AdamW([p.clone() for p in ps], state_bits=bits, max_grad_norm=0.1, device_step=True, **HYPER)
    held = [g.clone() for g in gs]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dev.step(held)
    assert int(dev.step_dev) == 0  # a capture runs nothing
    for t in range(4):
        new = _tensors([1000, 257], [F32], 30 * t)[1]
        for h, g in zip(held, new):
            h.copy_(g)
        graph.replay()
        eager.step(new)
    assert int(dev.step_dev) == 4
    assert all(torch.equal(a, b) for a, b in zip(dev.params, eager.params))
    for sa, sb in zip(dev.state, eager.state):
        assert all(torch.equal(x, y) for x, y in zip(sa, sb))
    assert torch.equal(dev.norm, eager.norm)


def test_two_optimizers_at_once(cuda_device):
    sets = [_tensors([50000, 3], [BF16], s) for s in range(3)]
    want = []
    for ps, gs in sets:
        o = nn.AdamW([p.clone() for p in ps], state_bits=8, max_grad_norm=0.2, **HYPER)
        for _ in range(5):
            o.step(gs)
        want.append(o)
    torch.cuda.synchronize()
    opts = [nn.AdamW([p.clone() for p in ps], state_bits=8, max_grad_norm=0.2, **HYPER) for ps, _ in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        for o, (_, gs), s in zip(opts, sets, streams):
            o.step(gs, stream=s)
    torch.cuda.synchronize()
    for a, b in zip(opts, want):
        assert all(torch.equal(x, y) for x, y in zip(a.params, b.params))


def test_zero_gradients(cuda_device):
    """A value that never had a gradient only decays, in both kinds of state."""
    for bits in (32, 8):
        p = _randn(600, 1)
        p0 = p.clone()
        opt = nn.AdamW([p], state_bits=bits, lr=0.1, weight_decay=0.5)
        g = torch.zeros(600, device="cuda")
        g[300:] = 0.01
        for _ in range(3):
            opt.step([g])
        # three roundings a step
        want = p0[:300].double() * (1 - 0.1 * 0.5) ** 3
        assert ((p[:300].double() - want).abs() <= 9 * U * want.abs()).all()
        assert (p[300:] != p0[300:]).all()


def test_dead_gradients_stop_moving_8bit_values(cuda_device):
    """Where gradients stop, 8-bit first moments reach zero although others of
    their block go on, and the values then only decay."""
    p = torch.zeros(256, device="cuda")
    opt = nn.AdamW([p], state_bits=8, lr=0.01, betas=(0.5, 0.9), weight_decay=0.0)
    g = torch.full((256,), 1.0, device="cuda")
    opt.step([g])
    g[:128] = 0
    for _ in range(40):
        opt.step([g])
    assert (opt.state[0][0][:128] == 0).all() and (opt.state[0][2][:128] > 0).all()
    before = p[:128].clone()
    opt.step([g])
    assert torch.equal(p[:128], before)


@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_that_are_not_finite(cuda_device, bits):
    """They reach their own value at once and nothing outside their block."""
    for bad in (float("inf"), float("nan")):
        ps, gs = _tensors([1000], [F32])
        ref = nn.AdamW([ps[0].clone()], state_bits=bits, **HYPER)
        ref.step(gs)
        g = gs[0].clone()
        g[300] = bad
        opt = nn.AdamW([ps[0].clone()], state_bits=bits, **HYPER)
        opt.step([g])
        ok = torch.arange(1000, device="cuda") != 300
        assert torch.equal(opt.params[0][ok], ref.params[0][ok]) and opt.params[0][300].isnan()
        if bits == 8:
            for s in (1, 3):
                assert opt.state[0][s].isnan().tolist() == [False, True, False, False]
            vals = ops.adamw_state_values(opt.state[0][0], opt.state[0][1])
            assert vals[256:512].isnan().all() and vals[:256].isfinite().all()


def test_state_values(cuda_device):
    ps, gs = _tensors([1, 255, 4000], [F32])
    opt = nn.AdamW(ps, state_bits=8, **HYPER)
    opt.step(gs)
    for mq, ms, vq, vs in opt.state:
        m, v = ops.adamw_state_values(mq, ms), ops.adamw_state_values(vq, vs)
        assert m.dtype is BF16 and m.shape == mq.shape
        for got, want in ((m, _decode(mq, ms)), (v, _decode(vq, vs))):
            # half a step, and four roundings of float32
            assert ((got.double() - want).abs() <= (2.0 ** -8 + 8 * U) * want.abs()).all()
    odd = torch.zeros(4001, device="cuda", dtype=torch.int8)[1:]
    odd.copy_(opt.state[2][0])
    assert torch.equal(ops.adamw_state_values(odd, opt.state[2][1]),
                       ops.adamw_state_values(opt.state[2][0], opt.state[2][1]))


def test_refusals(cuda_device):
    ps, gs = _tensors([300, 40], [F32])
    with pytest.raises(TypeError):
        nn.AdamW([p.to(BF16) for p in ps])
    with pytest.raises(ValueError):
        nn.AdamW([ps[0][::2]])
    with pytest.raises(ValueError):
        nn.AdamW(ps, copies=[None])
    with pytest.raises(TypeError):
        nn.AdamW(ps, copies=[ps[0], None])
    with pytest.raises(ValueError):
        nn.AdamW(ps, weight_decay=[0.1])
    with pytest.raises(ValueError):
        nn.AdamW(ps, state=[(ps[0], ps[0])])
    with pytest.raises(ValueError):
        nn.AdamW(ps, state=[(p, p, p) for p in ps])
    with pytest.raises(ValueError):
        nn.AdamW(ps, state=[(ps[1], ps[1]), (ps[1], ps[1])])
    with pytest.raises(TypeError):
        nn.AdamW(ps, state_bits=8, state=[(p, p, p, p) for p in ps])
    opt = nn.AdamW(ps)
    with pytest.raises(ValueError):
        opt.step(gs[:1])
    with pytest.raises(TypeError):
        opt.step([gs[0].half(), gs[1]])
    with pytest.raises(ValueError):
        opt.step([gs[1], gs[0]])
    with pytest.raises(ValueError):
        opt.step([torch.zeros(600, device="cuda")[::2], gs[1]])
    assert opt.step_count == 0
    for bad in (dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1.0), dict(max_grad_norm=-1.0)):
        with pytest.raises(_lib.MXError, match="invalid argument"):
            nn.AdamW(ps, **bad).step(gs)
    with pytest.raises(_lib.MXError, match="invalid argument"):
        nn.AdamW(ps, step_count=-1).step(gs)
    q = torch.zeros(300, device="cuda", dtype=torch.uint8)
    with pytest.raises(TypeError):
        ops.adamw_state_values(ps[0], torch.zeros(2, device="cuda"))
    with pytest.raises(ValueError):
        ops.adamw_state_values(q, torch.zeros(1, device="cuda"))
    L, h = _lib.lib(), ops.context(0)
    t = (_lib.AdamWTensor * 1)()
    t[0].param = t[0].grad = t[0].m = t[0].v = ps[0].data_ptr()
    t[0].n, t[0].grad_type = 300, 5
    bad = _lib.MX_ERR_INVALID
    args = (1e-3, 0.9, 0.99, 1e-8, 1, None, 0.0, None, None, 0, None)
    assert L.mx_adamw_step(h, t, 1, 32, *args) == bad  # an unknown type
    t[0].grad_type = 0
    assert L.mx_adamw_step(h, t, 1, 8, *args) == bad   # no scales
    assert L.mx_adamw_step(h, t, 1, 16, *args) == bad
    assert L.mx_adamw_step(h, None, 1, 32, *args) == bad
    t[0].n = -1
    assert L.mx_adamw_step(h, t, 1, 32, *args) == bad
    t[0].n = 300
    assert L.mx_adamw_step(h, t, 1, 32, 1e-3, 0.9, 0.99, 1e-8, 1, None, 1.0, None, None, 0, None) == bad


def test_memory_that_moved_is_refused(cuda_device):
    """The optimizer holds addresses: a parameter that was given other memory is
    an error, and nothing is written to the old."""
    p, g = torch.ones(300, device="cuda"), torch.ones(300, device="cuda")
    old = p.detach()
    opt = nn.AdamW([p], **HYPER)
    opt.step([g])
    before = old.clone()
    p.data = torch.zeros(300, device="cuda")
    with pytest.raises(ValueError, match="other memory"):
        opt.step([g])
    assert torch.equal(old, before) and (p == 0).all() and opt.step_count == 1
    again = nn.AdamW([p], state=opt.state, step_count=opt.step_count, **HYPER)
    again.step([g])
    assert (p != 0).all() and again.step_count == 2


def test_step_count_on_the_device_is_the_devices(cuda_device):
    p, g = torch.ones(300, device="cuda"), torch.ones(300, device="cuda")
    opt = nn.AdamW([p], device_step=True, step_count=5, **HYPER)
    opt.step([g])
    assert opt.step_count == 6
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step([g])
    assert opt.step_count == 6  # a capture runs nothing
    for _ in range(3):
        graph.replay()
    assert opt.step_count == 9


def test_shared_memory_is_refused(cuda_device):
    p = torch.ones(600, device="cuda")
    with pytest.raises(ValueError, match="share memory"):
        nn.AdamW([p, p])
    with pytest.raises(ValueError, match="share memory"):
        nn.AdamW([p[:400], p[300:]])
    m = torch.zeros(600, device="cuda")
    with pytest.raises(ValueError, match="share memory"):
        nn.AdamW([p], state=[(m, m)])
    nn.AdamW([p[:300], p[300:]]).step([torch.ones(300, device="cuda")] * 2)


def test_step_on_another_stream(cuda_device):
    p = torch.ones(5000, device="cuda")
    ref = p.clone()
    g = torch.linspace(-1, 1, 5000, device="cuda")
    s = torch.cuda.Stream()
    a = nn.AdamW([p], max_grad_norm=0.5, **HYPER)
    s.wait_stream(torch.cuda.current_stream())
    a.step([g], stream=s)
    torch.cuda.current_stream().wait_stream(s)
    b = nn.AdamW([ref], max_grad_norm=0.5, **HYPER)
    b.step([g])
    assert torch.equal(p, ref) and torch.equal(a.norm, b.norm)
