"""GPU tests of the gated linear layer (ops.gated_linear,
ops.gated_linear_backward) against a plain implementation in 64 bits.

Tolerances, value by value.  A product of depth K on the tensor cores adds K / 16
truncated partial sums (one unit in the last place, 2^-23, of the running sum
each), on the SIMT kernels at most K rounded ones; three-copy products drop
terms below 3 * 2^-24 and add K / 64 chunks of at most 24 truncations.  So g and
u are off by less than E = (K / 16 + 40) 2^-23 (K for SIMT) sum |x||w|.  The
activations' derivatives are below 1.2 and their second derivatives below 1.2,
their evaluation is good to 16 units in the last place of max(1, |z|).  dpre is
rounded to bfloat16 once for bfloat16 tensors (2^-8), and each stored value once
more.
"""
from __future__ import annotations

import math

import pytest
import torch

from moonxi_net_b200 import _lib, ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16
ACTS = ["silu", "gelu", "gelu_tanh", "relu", "sigmoid"]


def _half(t):
    return torch.finfo(t).eps / 2


def _act(name, z):
    """(act, derivative) in 64 bits."""
    s = torch.sigmoid(z)
    if name == "silu":
        return z * s, s * (1 + z * (1 - s))
    if name == "gelu":
        c = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * c, c + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        k = math.sqrt(2 / math.pi)
        t = torch.tanh(k * (z + 0.044715 * z ** 3))
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * k * (1 + 3 * 0.044715 * z * z)
    if name == "relu":
        return z.clamp_min(0), (z > 0).double()
    return s, s * (1 - s)


def _problem(M, K, F, dtype, tw, bias, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)

    def randn(*s):
        return torch.randn(*s, device="cuda", generator=g)
    w = randn(2 * F, K) if tw else randn(K, 2 * F)
    return (randn(M, K).to(dtype), (w / max(K, 1) ** 0.5).to(dtype),
            (0.3 * randn(2 * F)).to(dtype) if bias else None, randn(M, F).to(dtype))


def _check(name, got, ref, tol):
    lim = tol + _half(got.dtype) * ref.abs() + 1e-38
    ratio = ((got.double() - ref).abs() / lim)
    assert not (ratio > 1).any() and not ratio.isnan().any(), (name, float(ratio.max()))


def _halves(pre, F):
    p = pre.shape[-1] // 2
    return torch.cat((pre[..., :F], pre[..., p:p + F]), -1)


def _run_and_check(M, K, F, dtype, tw, act, bias, precision="default", seed=0):
    x, w, b, dh = _problem(M, K, F, dtype, tw, bias, seed)
    h, pre = ops.gated_linear(x, w, b, act=act, transpose_w=tw, save=True, precision=precision)
    dx, dw, db = ops.gated_linear_backward(dh, pre, x, w, act=act, transpose_w=tw,
                                           want_bias=bias, precision=precision)
    X, W, D = x.double(), w.double().t() if tw else w.double(), dh.double()
    B = b.double() if bias else torch.zeros(2 * F, device="cuda", dtype=torch.double)
    P = X @ W + B
    depth = K if dtype is F32 else K / 16  # SIMT's is the larger bound
    E = (depth + 40) * 2.0 ** -23 * (X.abs() @ W.abs() + B.abs())
    g, u, eg, eu = P[:, :F], P[:, F:], E[:, :F], E[:, F:]
    a, da = _act(act, g)
    small = 32 * U * g.abs().clamp_min(1)  # 16 units of an evaluation
    ea = 1.2 * eg + small
    _check("pre", _halves(pre, F), P, E)
    _check("h", h, a * u, ea * u.abs() + a.abs() * eu + ea * eu + 2 * U * (a * u).abs())
    # the derivative jumps at 0 for ReLU: where g is that close, either side
    jump = (g.abs() <= eg).double() if act == "relu" else 0.0
    eda = 1.2 * eg + small + jump
    rnd = _half(dtype) if dtype is BF16 else 4 * U
    dg, du = D * u * da, D * a
    edg = D.abs() * (eu * da.abs() + u.abs() * eda + eu * eda) + rnd * dg.abs()
    edu = D.abs() * ea + rnd * du.abs()
    dp, ep = torch.cat((dg, du), 1), torch.cat((edg, edu), 1)
    d2 = (2 * F if dtype is F32 else F / 8) + 40
    _check("dx", dx, dp @ W.t(), ep @ W.t().abs() + d2 * 2.0 ** -23 * (dp.abs() + ep) @ W.t().abs())
    dm = (M if dtype is F32 else M / 16) + 40
    ref, tol = X.t() @ dp, X.t().abs() @ ep + dm * 2.0 ** -23 * X.t().abs() @ (dp.abs() + ep)
    _check("dw", dw, ref.t() if tw else ref, tol.t() if tw else tol)
    if bias:  # summed before dpre is rounded
        _check("dbias", db, dp.sum(0), ep.sum(0) + 96 * U * dp.abs().sum(0))
    else:
        assert db is None
    status = ops.status()
    assert status == (0, 0)


# (M, K, F): single tokens, rows that split K, one tile and its edges, several
# tiles, widths off 8, 16 and 32
SHAPES = [(1, 64, 8), (1, 1000, 264), (2, 9, 5), (3, 2049, 24), (4, 520, 1000), (5, 4096, 40),
          (7, 1, 1), (24, 333, 64), (33, 77, 45), (64, 1024, 200), (128, 64, 128), (129, 65, 129),
          (256, 128, 136), (257, 200, 16), (300, 999, 40), (515, 333, 1001), (1000, 72, 300)]


@pytest.mark.parametrize("tw", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M,K,F", SHAPES)
def test_against_64_bits(cuda_device, M, K, F, dtype, tw):
    act = ACTS[(M + K + F) % len(ACTS)]
    _run_and_check(M, K, F, dtype, tw, act, bias=(M + F) % 2 == 0, seed=M + K)


@pytest.mark.parametrize("tw", [False, True])
@pytest.mark.parametrize("K,F", [(1024, 4096), (1000, 4099)])
def test_many_tiles(cuda_device, K, F, tw):
    """Rows for several of a pair's larger tiles, the last one in part; with and
    without pre, which the choice of tiles depends on."""
    M = 2125
    _run_and_check(M, K, F, BF16, tw, "silu", not tw, seed=K)
    x, w, b, _ = _problem(M, K, F, BF16, tw, not tw, seed=K)
    h, pre = ops.gated_linear(x, w, b, transpose_w=tw)
    assert pre is None
    P = x.double() @ (w.double().t() if tw else w.double()) + (b.double() if b is not None else 0)
    E = (K / 16 + 40) * 2.0 ** -23 * (x.double().abs() @ (w.t() if tw else w).double().abs()
                                     + (b.double().abs() if b is not None else 0))
    g, u, eg, eu = P[:, :F], P[:, F:], E[:, :F], E[:, F:]
    a = _act("silu", g)[0]
    ea = 1.2 * eg + 32 * U * g.abs().clamp_min(1)
    _check("h", h, a * u, ea * u.abs() + a.abs() * eu + ea * eu + 2 * U * (a * u).abs())


# few rows: lengths on both sides of each of their kernels' widths and splits,
# rows that start on any element
@pytest.mark.parametrize("tw", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("K,F", [(1, 1), (3, 2), (7, 9), (9, 3), (255, 257), (1025, 1151),
                                 (2051, 2369), (4099, 127), (130, 4741)])
def test_few_rows(cuda_device, K, F, dtype, tw):
    for M in (1, 2, 3, 4):
        _run_and_check(M, K, F, dtype, tw, ACTS[(M + K) % len(ACTS)], M % 2 == 0, seed=M + F)


@pytest.mark.parametrize("tw", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_few_rows_at_any_address(cuda_device, dtype, tw):
    """The products of aligned tensors and of copies that start 1 to 7 elements
    in, between values that would spoil a sum they get into."""
    for K, F in ((64, 40), (61, 37), (2048, 24)):
        for M in (1, 2, 4):
            x, w, b, _ = _problem(M, K, F, dtype, tw, True, seed=K + M)
            P = x.double() @ (w.double().t() if tw else w.double()) + b.double()
            tol = (K + 40) * 2.0 ** -23 * (x.double().abs() @ (w.double().t() if tw else w.double()).abs()
                                           + b.double().abs())
            for off in range(8):
                def moved(t):
                    buf = torch.full((t.numel() + 16,), math.nan, device="cuda", dtype=dtype)
                    v = buf[off:off + t.numel()].view(t.shape)
                    v.copy_(t)
                    return v
                _, pre = ops.gated_linear(moved(x), moved(w), moved(b), transpose_w=tw, save=True)
                _check("pre", _halves(pre, F), P, tol)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype,precision", [(BF16, "default"), (F32, "fp32"), (F32, "3xtf32"),
                                             (F32, "nparray")])
def test_activations_and_precisions(cuda_device, act, dtype, precision):
    for M in (3, 40, 200):
        _run_and_check(M, 96, 72, dtype, M == 40, act, True, precision)


def test_float32_tensor_products_keep_float32(cuda_device):
    """Large float32 products leave the exact kernels; their error stays at
    float32's: each of the K / 64 chunks is truncated at most 24 times (the
    last four at full size) and rounded once, relatively 2^-23 of the chunk, and
    chunks add up like a random walk: below 8 * 2^-24 of sqrt(sum (x w)^2)-sized
    results; held to 1e-6 of the norm."""
    x, w, _, dh = _problem(512, 1024, 2048, F32, False, False)
    h, pre = ops.gated_linear(x, w, save=True)
    P = x.double() @ w.double()
    assert float((_halves(pre, 2048).double() - P).norm() / P.norm()) < 1e-6
    exact = ops.gated_linear(x, w, precision="fp32")[0]
    assert not torch.equal(exact, h)  # two kernels


@pytest.mark.parametrize("M", [40, 300])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_unaligned_tensors(cuda_device, dtype, M):
    """Views that start off 16 bytes give what aligned copies give: the same
    bits on the tensor cores, whose sums do not depend on the alignment; on the
    SIMT kernels (40 float32 rows) the order of sums does, so there two results
    that are each off by at most depth * 2^-24 of their terms' sum."""
    x, w, b, dh = _problem(M, 64, 48, dtype, False, True)
    want_h, want_pre = ops.gated_linear(x, w, b, save=True)
    want = ops.gated_linear_backward(dh, want_pre, x, w)
    simt = dtype is F32 and M == 40

    def off(t):
        v = torch.empty(t.numel() + 1, device="cuda", dtype=dtype)[1:].view(t.shape)
        v.copy_(t)
        return v
    xo, wo, bo, do = off(x), off(w), off(b), off(dh)
    h, pre = ops.gated_linear(xo, wo, bo, save=True, out=off(want_h))
    got = ops.gated_linear_backward(do, want_pre, xo, wo, dx=off(want[0]), dw=off(want[1]))
    if simt:
        X, W, B = x.double().abs(), w.double().abs(), b.double().abs()
        E = 2 * (64 + 2) * U * (X @ W + B)
        _check("pre", _halves(pre, 48), _halves(want_pre, 48).double(), E)
        g, u = _halves(want_pre, 48).double().chunk(2, 1)
        small = 64 * U * g.abs().clamp_min(1)
        a = _act("silu", g)[0].abs()
        _check("h", h, want_h.double(), (1.2 * E[:, :48] + small) * (u.abs() + E[:, 48:]) + a * E[:, 48:])
        D = dh.double().abs()
        dp = torch.cat((D * u.abs() * 1.2, D * a), 1)  # the same dpre on both sides
        _check("dx", got[0], want[0].double(), 2 * (96 + 2) * U * dp @ W.t())
        _check("dw", got[1], want[1].double(), 2 * (40 + 2) * U * X.t() @ dp)
        assert torch.equal(got[2], want[2])
    else:
        for a, c in zip((h, pre, *got), (want_h, want_pre, *want)):
            assert torch.equal(a, c)
    # one to four rows
    h1 = ops.gated_linear(xo[:3].contiguous(), wo, bo)[0]
    _check("h", h1, want_h[:3].double(), 2 * _half(dtype) * want_h[:3].double().abs() + 1e-5)


def test_leading_dimensions(cuda_device):
    x, w, b, dh = _problem(24, 96, 40, BF16, False, True)
    h, pre = ops.gated_linear(x, w, b, save=True)
    h3, pre3 = ops.gated_linear(x.view(2, 12, 96), w, b, save=True)
    assert h3.shape == (2, 12, 40) and torch.equal(h3.view(24, 40), h)
    dx3, dw3, db3 = ops.gated_linear_backward(dh.view(2, 12, 40), pre3, x.view(2, 12, 96), w)
    dx, dw, db = ops.gated_linear_backward(dh, pre, x, w)
    assert torch.equal(dx3.view(24, 96), dx) and torch.equal(dw3, dw) and torch.equal(db3, db)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_empty_and_depthless(cuda_device, dtype):
    x, w, b, dh = _problem(0, 16, 24, dtype, False, True)
    h, pre = ops.gated_linear(x, w, b, save=True)
    assert h.shape == (0, 24)
    dx, dw, db = ops.gated_linear_backward(dh, pre, x, w)
    assert dx.shape == (0, 16) and (dw == 0).all() and (db == 0).all()
    # no features: [g | u] is the bias
    x, w, b, dh = _problem(5, 0, 24, dtype, False, True)
    h, pre = ops.gated_linear(x, w, b, save=True)
    B = b.double()
    assert torch.equal(_halves(pre, 24), b.float().expand(5, 48))
    want = _act("silu", B[:24])[0] * B[24:]
    _check("h", h, want.expand(5, 24), 32 * U * want.abs().expand(5, 24))
    dx, dw, db = ops.gated_linear_backward(dh, pre, x, w)
    assert dx.shape == (5, 0) and dw.shape == (0, 48)
    a, da = _act("silu", B[:24])
    dp = torch.cat((dh.double() * B[24:] * da, dh.double() * a), 1)
    _check("dbias", db, dp.sum(0), 96 * U * dp.abs().sum(0) + 64 * U * dh.double().abs().sum(0).repeat(2))


def test_nothing_beside_the_outputs_is_written(cuda_device):
    for M, K, F, dtype in ((3, 64, 24, BF16), (40, 64, 37, BF16), (300, 64, 37, F32), (9, 16, 8, F32)):
        x, w, b, dh = _problem(M, K, F, dtype, False, True)
        pre = ops.gated_linear(x, w, b, save=True)[1]

        def guarded(*shape):
            n = math.prod(shape)
            buf = torch.full((n + 128,), 5.0, device="cuda", dtype=dtype)
            return buf, buf[64:64 + n].view(shape)
        bufs = [guarded(M, F), guarded(M, K), guarded(K, 2 * F), guarded(2 * F)]
        ops.gated_linear(x, w, b, out=bufs[0][1])
        ops.gated_linear_backward(dh, pre, x, w, dx=bufs[1][1], dw=bufs[2][1], dbias=bufs[3][1])
        for buf, _ in bufs:
            assert (buf[:64] == 5.0).all() and (buf[-64:] == 5.0).all()


def test_rows_are_independent_of_what_is_not_finite(cuda_device):
    """A row that is not finite stays in its row of h and dx."""
    for M in (4, 40, 300):
        x, w, b, dh = _problem(M, 64, 48, BF16, False, True)
        h, pre = ops.gated_linear(x, w, b, save=True)
        dx = ops.gated_linear_backward(dh, pre, x, w)[0]
        x2 = x.clone()
        x2[1, 3] = float("nan")
        h2, pre2 = ops.gated_linear(x2, w, b, save=True)
        dx2 = ops.gated_linear_backward(dh, pre2, x2, w)[0]
        keep = [i for i in range(M) if i != 1]
        assert torch.equal(h2[keep], h[keep]) and h2[1].isnan().all()
        assert torch.equal(dx2[keep], dx[keep]) and dx2[1].isnan().all()


def test_large_pre_activations(cuda_device):
    """Exponentials that overflow or vanish leave the activations' limits."""
    x = torch.tensor([[200.0], [-200.0], [89.0], [-89.0], [0.0]], device="cuda")
    w = torch.tensor([[1.0, 1.0]], device="cuda")  # g = u = x
    for act in ACTS:
        h, pre = ops.gated_linear(x, w, act=act, save=True)
        a, da = _act(act, x.double())
        _check(act, h, a * x.double(), 64 * U * x.double().abs() ** 2 + 1e-35)
        dx = ops.gated_linear_backward(torch.ones_like(h), pre, x, w, act=act)[0]
        _check(act, dx, x.double() * da + a, 256 * U * x.double().abs().clamp_min(1) ** 2)


def test_gradient_against_differences(cuda_device):
    for act in ("silu", "gelu", "gelu_tanh", "sigmoid"):
        x, w, b, dh = _problem(9, 20, 12, F32, False, True, 3)
        pre = ops.gated_linear(x, w, b, act=act, save=True)[1]
        grads = ops.gated_linear_backward(dh, pre, x, w, act=act)
        g = torch.Generator("cuda").manual_seed(2)
        dirs = [torch.randn(t.shape, device="cuda", generator=g, dtype=torch.double) for t in (x, w, b)]

        def loss(e):
            xx, ww, bb = (t.double() + e * d for t, d in zip((x, w, b), dirs))
            P = xx @ ww + bb
            return (_act(act, P[:, :12])[0] * P[:, 12:] * dh.double()).sum()
        e = 1e-5
        diff = float((loss(e) - loss(-e)) / (2 * e))
        form = sum(float((t.double() * d).sum()) for t, d in zip(grads, dirs))
        scale = sum(float((t.double() * d).abs().sum()) for t, d in zip(grads, dirs))
        assert abs(diff - form) <= scale * (256 * U + 1e-7)


def test_repeats_streams_and_capture(cuda_device):
    """The same bits every time, on any stream, two calls at once, replayed."""
    for M, dtype in ((3, BF16), (64, BF16), (300, BF16), (20, F32), (300, F32)):
        x, w, b, dh = _problem(M, 1024, 136, dtype, False, True)

        def call(stream=None):
            h, pre = ops.gated_linear(x, w, b, save=True, stream=stream)
            return (h, pre, *ops.gated_linear_backward(dh, pre, x, w, stream=stream))
        want = call()
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(3)]
        got = [call(s) for _ in range(5) for s in streams]
        torch.cuda.synchronize()
        for t in got:
            assert all(torch.equal(p, q) for p, q in zip(want, t))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        for seed in (1, 2):
            x2 = _problem(M, 1024, 136, dtype, False, True, seed)[0]
            keep, x0 = x.clone(), x
            x0.copy_(x2)
            graph.replay()
            want2 = call()
            assert all(torch.equal(p, q) for p, q in zip(want2, out))
            x0.copy_(keep)


def test_only_some_gradients(cuda_device):
    x, w, b, dh = _problem(40, 64, 48, BF16, False, True)
    pre = ops.gated_linear(x, w, b, save=True)[1]
    want = ops.gated_linear_backward(dh, pre, x, w)
    L, h = _lib.lib(), ops.context(0)
    nb = L.mx_gated_linear_workspace_bytes(h, 1, 40, 64, 48, 0, 0, 1)
    ws = torch.empty(nb, dtype=torch.uint8, device="cuda")
    s = torch.cuda.current_stream().cuda_stream
    for only in range(3):
        out = torch.empty_like(want[only])
        ptrs = [out.data_ptr() if i == only else None for i in range(3)]
        rc = L.mx_gated_linear_bwd(h, 1, dh.data_ptr(), pre.data_ptr(), x.data_ptr(), w.data_ptr(),
                                   *ptrs, 40, 64, 48, 0, 0, 0, ws.data_ptr(), nb, s)
        assert rc == 0
        _check(str(only), out, want[only].double(), _half(BF16) * want[only].double().abs() + 1e-3)


def test_a_wait_that_gives_up_is_reported(cuda_device):
    """A wait limit of a nanosecond runs out at once: the call records it in the
    status word, and the context goes on."""
    ctx = ops.new_context(0)
    try:
        x, w, _, dh = _problem(300, 512, 256, BF16, False, False)
        want = ops.gated_linear(x, w, ctx=ctx)[0].clone()
        assert ops.context_status(ctx) == (0, 0)
        assert _lib.lib().mx_context_set_timeout_ns(ctx, 1) == 0
        ops.gated_linear(x, w, ctx=ctx)
        rc, where = ops.context_status(ctx)
        assert rc == _lib.MX_ERR_TIMEOUT and 400 < where < 410
        assert _lib.lib().mx_context_set_timeout_ns(ctx, 2_000_000_000) == 0
        assert torch.equal(ops.gated_linear(x, w, ctx=ctx)[0], want)
        assert ops.context_status(ctx) == (0, 0)
    finally:
        ops.destroy_context(ctx)


def test_refusals(cuda_device):
    x, w, b, dh = _problem(8, 32, 24, BF16, False, True)
    h, pre = ops.gated_linear(x, w, b, save=True)
    with pytest.raises(ValueError, match="act must be one of"):
        ops.gated_linear(x, w, act="tanh")
    with pytest.raises(TypeError):
        ops.gated_linear(x.half(), w.half())
    with pytest.raises(TypeError):
        ops.gated_linear(x, w.float())
    with pytest.raises(TypeError):
        ops.gated_linear(x, w, b.float())
    with pytest.raises(ValueError):
        ops.gated_linear(x, w.t())
    with pytest.raises(ValueError):
        ops.gated_linear(x, w[:, :47].contiguous())
    with pytest.raises(ValueError):
        ops.gated_linear(x[:, :16], w)
    with pytest.raises(ValueError):
        ops.gated_linear(x[:, ::2], w[:16])
    with pytest.raises(ValueError):
        ops.gated_linear(x, w, b[:24])
    with pytest.raises(ValueError):
        ops.gated_linear(x, w, out=torch.empty(8, 25, device="cuda", dtype=BF16))
    with pytest.raises(ValueError):
        ops.gated_linear_backward(dh[:4], pre, x, w)
    with pytest.raises(ValueError):
        ops.gated_linear_backward(dh, pre[:, :24].contiguous(), x, w)
    with pytest.raises(TypeError):
        ops.gated_linear_backward(dh, pre.to(BF16), x, w)
    L, hd = _lib.lib(), ops.context(0)
    bad = _lib.MX_ERR_INVALID
    p = [t.data_ptr() for t in (x, w, h)]
    x40 = torch.zeros(40, 33, device="cuda", dtype=BF16)
    need = L.mx_gated_linear_workspace_bytes(hd, 1, 40, 33, 24, 0, 0, 0)
    assert need > 0  # rows of 66 bytes are packed
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    big = torch.zeros(40, 48, device="cuda", dtype=BF16)
    call = (hd, 1, x40.data_ptr(), big.data_ptr(), None, big.data_ptr(), None, 40, 33, 24, 0)
    assert L.mx_gated_linear_fwd(*call, 0, 0, ws.data_ptr(), need - 1, None) == bad
    assert L.mx_gated_linear_fwd(*call, 0, 0, None, need, None) == bad
    assert L.mx_gated_linear_fwd(*call, 5, 0, ws.data_ptr(), need, None) == bad
    assert L.mx_gated_linear_fwd(*call, 0, 9, ws.data_ptr(), need, None) == bad
    assert L.mx_gated_linear_fwd(hd, 7, *call[2:], 0, 0, ws.data_ptr(), need, None) == bad
    assert L.mx_gated_linear_fwd(hd, 1, p[0], p[1], None, p[2], pre.data_ptr() + 4, 8, 32, 24, 0, 0,
                                 0, None, 0, None) == bad  # pre off 32 bytes
    assert L.mx_gated_linear_fwd(hd, 1, None, p[1], None, p[2], None, 8, 32, 24, 0, 0, 0, None, 0,
                                 None) == bad


def test_shared_memory_and_sizes_are_refused(cuda_device):
    x, w, b, dh = _problem(8, 24, 24, BF16, False, True)
    h, pre = ops.gated_linear(x, w, b, save=True)
    with pytest.raises(ValueError, match="share memory"):
        ops.gated_linear(x, w, b, out=x)
    with pytest.raises(ValueError, match="share memory"):
        ops.gated_linear_backward(dh, pre, x, w, dx=x)
    with pytest.raises(ValueError, match="share memory"):
        ops.gated_linear_backward(dh, pre, x, w, dw=w)
    both = torch.empty(2 * 8 * 24, device="cuda", dtype=BF16)  # out and x overlap in part
    with pytest.raises(ValueError, match="share memory"):
        ops.gated_linear(both[:192].view(8, 24), w, b, out=both[100:292].view(8, 24))
    ops.gated_linear(both[:192].view(8, 24), w, b, out=both[192:].view(8, 24))
    L, hd = _lib.lib(), ops.context(0)
    p = [t.data_ptr() for t in (x, w, h)]
    for m, k, f in ((2 ** 31 - 1, 24, 24), (8, 2 ** 31 - 1, 24), (8, 24, 2 ** 30 - 1)):
        assert L.mx_gated_linear_fwd(hd, 1, p[0], p[1], None, p[2], None, m, k, f, 0, 0, 0, None, 0,
                                     None) == _lib.MX_ERR_UNSUPPORTED
        assert L.mx_gated_linear_workspace_bytes(hd, 1, m, k, f, 0, 0, 0) == 0


def test_long_and_thin(cuda_device):
    """A product over 42 million rows, whose whole cost in cycles passes 31 bits."""
    M, K, F = 42_000_001, 8, 8
    x = torch.full((M, K), 0.5, device="cuda")
    w = torch.zeros(K, 2 * F, device="cuda")
    b = torch.ones(2 * F, device="cuda")
    h, pre = ops.gated_linear(x, w, b, act="relu", save=True)
    assert (h == 1).all()
    dx, dw, db = ops.gated_linear_backward(h.mul_(0.25), pre, x, w, act="relu")
    assert (dx == 0).all()
    # dpre = 0.25 everywhere: dw = M / 8, db = M / 4, all of whose terms have one
    # sign: M / 64 rounded sums of k-blocks of at most 24 truncations, and sums of
    # no more terms than that for db
    tol = M / 64 * U + 24 * 2 * U
    assert ((dw.double() / (M / 8) - 1).abs() <= tol).all()
    assert ((db.double() / (M / 4) - 1).abs() <= tol).all()
