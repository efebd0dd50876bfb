"""Device ops of the matmul path, called through the C ABI.

torch is used only for device memory and streams: every function here takes
CUDA tensors (float32; the layer norm, gated layer and AdamW also bfloat16),
passes their raw pointers and the current torch stream to ``libmxgemm.so`` and
lets the library's kernels do the work.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from ._lib import PRECISIONS, check

_ctx_cache: dict[tuple, int] = {}


def context(device: int | None = None, mode: str = "default") -> int:
    """The library context (the ABI's ``handle``) for a device and precision
    mode, created once.  A context in "nparray" mode also runs the
    training-step ops in the NpArray CPU order (bit-identical results)."""
    if device is None:
        device = torch.cuda.current_device()
    key = (int(device), mode)
    h = _ctx_cache.get(key)
    if h is None:
        h = _lib.lib().mx_context_create(int(device))
        if not h:
            raise _lib.MXError(_lib.MX_ERR_NO_DEVICE, f"mx_context_create({device})")
        if mode != "default":
            check(_lib.lib().mx_context_set_precision(h, _prec(mode)), "mx_context_set_precision")
        _ctx_cache[key] = h
    return h


def new_context(device: int, mode: str = "default") -> int:
    """A context owned by the caller (not shared through `context`); free it
    with `destroy_context`."""
    h = _lib.lib().mx_context_create(int(device))
    if not h:
        raise _lib.MXError(_lib.MX_ERR_NO_DEVICE, f"mx_context_create({device})")
    if mode != "default":
        check(_lib.lib().mx_context_set_precision(h, _prec(mode)), "mx_context_set_precision")
    return h


def destroy_context(h) -> None:
    if h:
        _lib.lib().mx_context_destroy(h)


def set_sm_budget(ctx, sms: int) -> None:
    """SMs the context's tensor-core GEMMs prefer (0 = all); a launch takes
    every SM when that finishes it more than 3 % sooner."""
    check(_lib.lib().mx_context_set_sm_budget(ctx, int(sms)), "mx_context_set_sm_budget")


def set_sm_limit(ctx, sms: int) -> None:
    """Hard cap on the SMs of the context's tensor-core GEMMs (0 = none)."""
    check(_lib.lib().mx_context_set_sm_limit(ctx, int(sms)), "mx_context_set_sm_limit")


def _handle(ctx, t: torch.Tensor) -> int:
    return ctx if ctx is not None else context(t.device.index)


def _prec(precision) -> int:
    if isinstance(precision, str):
        return PRECISIONS[precision]
    return int(precision)


def _stream_ptr(stream=None) -> int:
    s = stream if stream is not None else torch.cuda.current_stream()
    return s.cuda_stream


def _check_tensor(t: torch.Tensor, name: str, numel: int | None = None):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor")
    if t.dtype != torch.float32:
        raise TypeError(f"{name} must be float32, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if numel is not None and t.numel() < numel:
        raise ValueError(f"{name} has {t.numel()} elements, needs {numel}")


def matmul(a: torch.Tensor, b: torch.Tensor, M: int, K: int, N: int, ta: bool = False,
           tb: bool = False, alpha: float = 1.0, beta: float = 0.0,
           out: torch.Tensor | None = None, precision="default", stream=None,
           ctx=None) -> torch.Tensor:
    """C[M,N] = alpha op(A) op(B) + beta C (the reference's cuda_matmul)."""
    _check_tensor(a, "a", M * K)
    _check_tensor(b, "b", K * N)
    if out is None:
        out = torch.empty((M, N), device=a.device, dtype=torch.float32)
    _check_tensor(out, "out", M * N)
    rc = _lib.lib().moonbit_cuda_matmul_ex(
        _handle(ctx, a), a.data_ptr(), b.data_ptr(), out.data_ptr(), M, K, N, int(ta),
        int(tb), float(alpha), float(beta), _stream_ptr(stream), _prec(precision))
    check(rc, "moonbit_cuda_matmul_ex")
    return out


def gemm(a: torch.Tensor, b: torch.Tensor, M: int, K: int, N: int, ta: bool = False,
         tb: bool = False, alpha: float = 1.0, beta: float = 0.0,
         bias: torch.Tensor | None = None, relu: bool = False,
         out: torch.Tensor | None = None, precision="default", stream=None,
         lda: int = 0, ldb: int = 0, ldc: int = 0, ctx=None) -> torch.Tensor:
    """C = act(alpha op(A) op(B) + beta C + bias) for any layout (mx_gemm_ex)."""
    _check_tensor(a, "a", M * K if not lda else 1)
    _check_tensor(b, "b", K * N if not ldb else 1)
    if bias is not None:
        _check_tensor(bias, "bias", N)
    if out is None:
        out = torch.empty((M, N), device=a.device, dtype=torch.float32)
    _check_tensor(out, "out", M * N if not ldc else 1)
    rc = _lib.lib().mx_gemm_ex(
        _handle(ctx, a), a.data_ptr(), b.data_ptr(), out.data_ptr(),
        bias.data_ptr() if bias is not None else None, M, K, N, int(ta), int(tb), int(lda),
        int(ldb), int(ldc), float(alpha), float(beta), int(relu), _stream_ptr(stream),
        _prec(precision))
    check(rc, "mx_gemm_ex")
    return out


def linear(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None, relu: bool = False,
           transpose_w: bool = False, out: torch.Tensor | None = None, alpha: float = 1.0,
           precision="default", stream=None, ctx=None) -> torch.Tensor:
    """y = act(alpha x op(w) + bias): w is [K,N] (transpose_w=False) or [N,K]."""
    M, K = x.shape
    N = w.shape[0] if transpose_w else w.shape[1]
    _check_tensor(x, "x")
    _check_tensor(w, "w", K * N)
    if bias is not None:
        _check_tensor(bias, "bias", N)
    if out is None:
        out = torch.empty((M, N), device=x.device, dtype=torch.float32)
    _check_tensor(out, "out", M * N)
    rc = _lib.lib().moonbit_cuda_linear_fwd_ex(
        _handle(ctx, x), x.data_ptr(), w.data_ptr(),
        bias.data_ptr() if bias is not None else None, out.data_ptr(), M, K, N,
        int(transpose_w), int(relu), float(alpha), _stream_ptr(stream), _prec(precision))
    check(rc, "moonbit_cuda_linear_fwd_ex")
    return out


def linear_bias_first(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor, relu: bool = True,
                      transpose_w: bool = True, out: torch.Tensor | None = None,
                      pre: torch.Tensor | None = None, stream=None, ctx=None):
    """The reference's fused_linear(_relu) (nparray/fused_ops.mbt:12-78): the
    sum starts from the bias, NpArray rounding order; returns (y, pre)."""
    M, K = x.shape
    N = w.shape[0] if transpose_w else w.shape[1]
    _check_tensor(x, "x")
    _check_tensor(w, "w", K * N)
    _check_tensor(bias, "bias", N)
    if out is None:
        out = torch.empty((M, N), device=x.device, dtype=torch.float32)
    _check_tensor(out, "out", M * N)
    if pre is not None:
        _check_tensor(pre, "pre", M * N)
    rc = _lib.lib().mx_linear_fwd_bias_first(
        _handle(ctx, x), x.data_ptr(), w.data_ptr(), bias.data_ptr(), out.data_ptr(),
        pre.data_ptr() if pre is not None else None, M, K, N, int(transpose_w), int(relu),
        _stream_ptr(stream))
    check(rc, "mx_linear_fwd_bias_first")
    return out, pre


def relu_backward(grad_out: torch.Tensor, saved: torch.Tensor, out: torch.Tensor | None = None,
                  stream=None, ctx=None) -> torch.Tensor:
    _check_tensor(grad_out, "grad_out")
    _check_tensor(saved, "saved", grad_out.numel())
    if out is None:
        out = torch.empty_like(grad_out)
    _check_tensor(out, "out", grad_out.numel())
    rc = _lib.lib().mx_relu_backward(_handle(ctx, grad_out), grad_out.data_ptr(),
                                     saved.data_ptr(), out.data_ptr(), grad_out.numel(),
                                     _stream_ptr(stream))
    check(rc, "mx_relu_backward")
    return out


def reduce_sum_leading(x: torch.Tensor, out: torch.Tensor | None = None,
                       stream=None, ctx=None) -> torch.Tensor:
    """Column sums of a [rows, cols] tensor (the bias gradient)."""
    rows, cols = x.shape
    _check_tensor(x, "x")
    if out is None:
        out = torch.empty((cols,), device=x.device, dtype=torch.float32)
    _check_tensor(out, "out", cols)
    rc = _lib.lib().mx_reduce_sum_leading(_handle(ctx, x), x.data_ptr(), out.data_ptr(),
                                          cols, rows, _stream_ptr(stream))
    check(rc, "mx_reduce_sum_leading")
    return out


def softmax_ce_labels(logits: torch.Tensor, labels: torch.Tensor, denom: int | None = None,
                      grad: torch.Tensor | None = None, loss: torch.Tensor | None = None,
                      want_grad: bool = True, stream=None, ctx=None):
    """(loss[1], dlogits) of mean cross-entropy with float class labels."""
    B, C = logits.shape
    _check_tensor(logits, "logits")
    _check_tensor(labels, "labels", B)
    if loss is None:
        loss = torch.empty((1,), device=logits.device, dtype=torch.float32)
    if want_grad and grad is None:
        grad = torch.empty_like(logits)
    rc = _lib.lib().mx_softmax_ce_labels(
        _handle(ctx, logits), logits.data_ptr(), labels.data_ptr(),
        grad.data_ptr() if want_grad else None, loss.data_ptr(), B, C,
        B if denom is None else int(denom), _stream_ptr(stream))
    check(rc, "mx_softmax_ce_labels")
    return loss, grad


def sgd_momentum_autoclip(params: torch.Tensor, grads: torch.Tensor, vels: torch.Tensor, lr: float,
                          momentum: float, weight_decay: float, max_grad_norm: float,
                          norm_out: torch.Tensor | None = None, n: int | None = None,
                          stream=None, ctx=None) -> None:
    n = params.numel() if n is None else n
    for t, name in ((params, "params"), (grads, "grads"), (vels, "vels")):
        _check_tensor(t, name, n)
    rc = _lib.lib().mx_sgd_momentum_autoclip(
        _handle(ctx, params), params.data_ptr(), grads.data_ptr(), vels.data_ptr(), n,
        float(lr), float(momentum), float(weight_decay), float(max_grad_norm),
        norm_out.data_ptr() if norm_out is not None else None, _stream_ptr(stream))
    check(rc, "mx_sgd_momentum_autoclip")


# ---------------------------------------------------------------- split form
def _ptr(t):
    return t.data_ptr() if t is not None else None


def split_tf32(src: torch.Tensor, hi: torch.Tensor, lo: torch.Tensor | None, ctx=None,
               stream=None) -> None:
    """hi/lo 3xTF32 split of a row-major 2-D (or flat, as one row) tensor."""
    _check_tensor(src, "src")
    rows, cols = (src.shape[0], src.shape[1]) if src.dim() == 2 else (1, src.numel())
    rc = _lib.lib().mx_split_tf32(_handle(ctx, src), src.data_ptr(), rows, cols, cols,
                                  hi.data_ptr(), _ptr(lo), cols, _stream_ptr(stream))
    check(rc, "mx_split_tf32")


def gemm_split(a_hi, a_lo, lda: int, a_kmajor: bool, b_hi, b_lo, ldb: int, b_kmajor: bool,
               M: int, K: int, N: int, c=None, c_hi=None, c_lo=None, ldc: int | None = None,
               alpha: float = 1.0, beta: float = 0.0, bias=None, relu: bool = False,
               mask=None, ldm: int = 0, passes: int = 3, padded: int = 0, ctx=None,
               stream=None, colsum=None, colsum_scratch=None) -> None:
    """tcgen05 GEMM on split operands (mx_gemm_split_ex); see the header.
    padded: bit 0 / bit 1 when A / B copies have 32 readable floats past
    their last row.  colsum: also write the column sums of the stored output
    (mx_gemm_split_colsum_ex; colsum_scratch holds colsum_scratch_bytes)."""
    ref = c if c is not None else c_hi
    args = (_handle(ctx, a_hi), a_hi.data_ptr(), _ptr(a_lo), lda, int(a_kmajor), b_hi.data_ptr(),
            _ptr(b_lo), ldb, int(b_kmajor), _ptr(c), _ptr(c_hi), _ptr(c_lo),
            N if ldc is None else ldc, M, K, N, float(alpha), float(beta), _ptr(bias), int(relu),
            _ptr(mask), ldm, passes, int(padded))
    if colsum is None:
        rc = _lib.lib().mx_gemm_split_ex(*args, _stream_ptr(stream))
        check(rc, "mx_gemm_split_ex")
    else:
        rc = _lib.lib().mx_gemm_split_colsum_ex(
            *args, colsum.data_ptr(), colsum_scratch.data_ptr(),
            colsum_scratch.numel() * colsum_scratch.element_size(), _stream_ptr(stream))
        check(rc, "mx_gemm_split_colsum_ex")
    return ref


def gemm_colsum_scratch_bytes(M: int, N: int) -> int:
    return int(_lib.lib().mx_gemm_colsum_scratch_bytes(M, N))


def _split_gemm(a_hi, a_lo, lda: int, a_kmajor: bool, b_hi, b_lo, ldb: int, b_kmajor: bool,
                M: int, K: int, N: int, c=None, c_hi=None, c_lo=None, ldc: int | None = None,
                alpha: float = 1.0, beta: float = 0.0, bias=None, relu: bool = False,
                mask=None, ldm: int = 0, padded: int = 0, colsum=None, colsum_scratch=None):
    g = _lib.SplitGemm()
    g.a_hi, g.a_lo, g.lda, g.a_kmajor = a_hi.data_ptr(), _ptr(a_lo), lda, int(a_kmajor)
    g.b_hi, g.b_lo, g.ldb, g.b_kmajor = b_hi.data_ptr(), _ptr(b_lo), ldb, int(b_kmajor)
    g.c, g.c_hi, g.c_lo = _ptr(c), _ptr(c_hi), _ptr(c_lo)
    g.ldc = N if ldc is None else ldc
    g.M, g.K, g.N, g.alpha, g.beta = M, K, N, float(alpha), float(beta)
    g.bias, g.relu, g.mask, g.ldm, g.flags = _ptr(bias), int(relu), _ptr(mask), ldm, int(padded)
    if colsum is not None:
        g.colsum, g.colsum_scratch = colsum.data_ptr(), colsum_scratch.data_ptr()
        g.colsum_scratch_bytes = colsum_scratch.numel() * colsum_scratch.element_size()
    return g


def gemm_split_pair(g0: dict, g1: dict, ctx=None, stream=None) -> None:
    """Two independent 3xTF32 split-operand GEMMs in one launch
    (mx_gemm_split_pair): each dict holds gemm_split's keyword arguments
    (a_hi ... colsum_scratch; passes is always 3)."""
    s0, s1 = _split_gemm(**g0), _split_gemm(**g1)
    rc = _lib.lib().mx_gemm_split_pair(_handle(ctx, g0["a_hi"]), ctypes.byref(s0),
                                       ctypes.byref(s1), _stream_ptr(stream))
    check(rc, "mx_gemm_split_pair")


def split_plan(M: int, N: int, K: int, passes: int = 3, ctx=None, device: int | None = None):
    """The work split the context's tcgen05 GEMM picks for M x N x K
    (mx_tc_split_plan): dict of mode (0 whole tiles, 1 stream-K, 2 tail
    split), tile0, r, kp, s, j."""
    out = (ctypes.c_int32 * 6)()
    h = ctx if ctx is not None else context(device)
    check(_lib.lib().mx_tc_split_plan(h, M, N, K, passes, out), "mx_tc_split_plan")
    return dict(zip(("mode", "tile0", "r", "kp", "s", "j"), (int(v) for v in out)))


def softmax_ce_colsum_scratch_bytes(batch: int, C: int) -> int:
    """0 when C is too large for the fused column sums."""
    return int(_lib.lib().mx_softmax_ce_colsum_scratch_bytes(batch, C))


def softmax_ce_labels_split(logits, labels, grad, g_hi, g_lo, loss, denom: int, ctx=None,
                            stream=None, colsum=None, colsum_scratch=None) -> None:
    """CE forward+backward writing the gradient and its split copy; with
    colsum, also the gradient's column sums (the output layer's bias
    gradient, mx_softmax_ce_labels_split_colsum)."""
    B, C = logits.shape
    if colsum is None:
        rc = _lib.lib().mx_softmax_ce_labels_split(
            _handle(ctx, logits), logits.data_ptr(), labels.data_ptr(), grad.data_ptr(),
            g_hi.data_ptr(), g_lo.data_ptr(), _ptr(loss), B, C, int(denom), _stream_ptr(stream))
        check(rc, "mx_softmax_ce_labels_split")
    else:
        rc = _lib.lib().mx_softmax_ce_labels_split_colsum(
            _handle(ctx, logits), logits.data_ptr(), labels.data_ptr(), grad.data_ptr(),
            g_hi.data_ptr(), g_lo.data_ptr(), _ptr(loss), B, C, int(denom), colsum.data_ptr(),
            colsum_scratch.data_ptr(), colsum_scratch.numel() * colsum_scratch.element_size(),
            _stream_ptr(stream))
        check(rc, "mx_softmax_ce_labels_split_colsum")


def sgd_momentum_autoclip_split(params, grads, vels, p_hi, p_lo, lr, momentum, weight_decay,
                                max_grad_norm, norm_out=None, ctx=None, stream=None) -> None:
    n = params.numel()
    rc = _lib.lib().mx_sgd_momentum_autoclip_split(
        _handle(ctx, params), params.data_ptr(), grads.data_ptr(), vels.data_ptr(), n,
        float(lr), float(momentum), float(weight_decay), float(max_grad_norm), _ptr(norm_out),
        p_hi.data_ptr(), p_lo.data_ptr(), _stream_ptr(stream))
    check(rc, "mx_sgd_momentum_autoclip_split")


def sum_squares(x, out, accumulate: bool = False, ctx=None, stream=None) -> None:
    """out[0] = (out[0] if accumulate else 0) + sum(x**2) (mx_sum_squares)."""
    rc = _lib.lib().mx_sum_squares(_handle(ctx, out), _ptr(x), x.numel(), out.data_ptr(),
                                   int(accumulate), _stream_ptr(stream))
    check(rc, "mx_sum_squares")


def sgd_momentum_clip(params, grads, vels, lr, momentum, weight_decay, max_grad_norm, norm_sq,
                      ctx=None, stream=None) -> None:
    """Momentum-SGD update of one range clipped by sqrt(norm_sq[0])
    (mx_sgd_momentum_clip)."""
    n = params.numel()
    rc = _lib.lib().mx_sgd_momentum_clip(
        _handle(ctx, params), params.data_ptr(), grads.data_ptr(), vels.data_ptr(), n,
        float(lr), float(momentum), float(weight_decay), float(max_grad_norm),
        norm_sq.data_ptr(), _stream_ptr(stream))
    check(rc, "mx_sgd_momentum_clip")


# ------------------------------ layer norm, the gated linear layer, AdamW
_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}


def _check_like(t: torch.Tensor, name: str, device: int, dtype, shape=None):
    """A contiguous CUDA tensor on the device `device`, of the given type."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor")
    if t.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.get_device() != device:
        raise ValueError(f"{name} is on cuda:{t.get_device()}, not on cuda:{device}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, needs {tuple(shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _check_type(t: torch.Tensor, name: str) -> int:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor")
    dt = _DTYPES.get(t.dtype)
    if dt is None:
        raise TypeError(f"{name} must be float32 or bfloat16, got {t.dtype}")
    return dt


def _launch_stream(device: int, stream) -> int:
    """The raw stream of a call: the given one, else the device's current one."""
    return stream.cuda_stream if stream is not None else \
        torch._C._cuda_getCurrentRawStream(device)


def _empty(shape, dtype, t, stream):
    """Memory on t's device for a call on `stream` (None: the current one),
    allocated on that stream, so that it is not handed on before the call is
    done with it.  (new_empty costs the host a quarter less than empty.)"""
    if stream is None:
        return t.new_empty(shape, dtype=dtype)
    with torch.cuda.stream(stream):
        return t.new_empty(shape, dtype=dtype)


def _empty_like(t, stream):
    """Memory for a tensor like a contiguous one (half the time of _empty)."""
    if stream is None:
        return torch.empty_like(t)
    with torch.cuda.stream(stream):
        return torch.empty_like(t)


_MAX_SIZE = 0x7FFF0000  # of a dimension


def _span(t: torch.Tensor) -> tuple[int, int, int, int]:
    """(address, bytes of a row, bytes from a row to the next, rows) of a
    contiguous tensor (one row) or a 2-D one with contiguous rows."""
    size = t.element_size()
    if t.is_contiguous():
        return t.data_ptr(), t.numel() * size, t.numel() * size, 1
    return t.data_ptr(), t.shape[1] * size, t.stride(0) * size, t.shape[0]


def _apart(out: torch.Tensor, name: str, *others) -> None:
    """An output that the caller gives does not share memory with what the call
    reads or writes beside it; rows may lie between another tensor's rows."""
    if not out.numel():
        return
    a, la, pa, na = _span(out)
    for t in others:
        if t is None or not t.numel():
            continue
        b, lb, pb, nb = _span(t)
        if b >= a + (na - 1) * pa + la or a >= b + (nb - 1) * pb + lb:
            continue
        if pa == pb and na > 1 and nb > 1:
            clear = la <= (b - a) % pa <= pa - lb
        else:  # row j ends behind another's row's start and starts before its end
            few, many = sorted(((a, la, pa, na), (b, lb, pb, nb)), key=lambda r: r[3])
            start = few[0] - many[0] + torch.arange(few[3]) * few[2]
            first = ((start - many[1]).div(many[2], rounding_mode="floor") + 1).clamp(min=0)
            last = -((-(start + few[1])).div(many[2], rounding_mode="floor")) - 1
            clear = not (first <= last.clamp(max=many[3] - 1)).any()
        if not clear:
            raise ValueError(f"{name} must not share memory with another argument")


def _rows(t: torch.Tensor, name: str) -> tuple[int, int, int]:
    """(rows, columns, row stride) of a tensor seen as rows of its last
    dimension: contiguous, or 2-D with contiguous rows."""
    if t.dim() < 1 or t.shape[-1] < 1:
        raise ValueError(f"{name} needs a last dimension of at least 1")
    cols = t.shape[-1]
    if cols > _MAX_SIZE or t.numel() > _MAX_SIZE * cols:
        raise ValueError(f"{name} has more than {_MAX_SIZE} rows or columns")
    if t.is_contiguous():
        return t.numel() // cols, cols, cols
    if t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= cols:
        return t.shape[0], cols, t.stride(0)
    raise ValueError(f"{name} must be contiguous, or 2-D with contiguous rows")


def _like_rows(t: torch.Tensor, name: str, x: torch.Tensor, of: str) -> int:
    """The row stride of a tensor of x's shape, type and device."""
    if not isinstance(t, torch.Tensor) or t.shape != x.shape or t.dtype is not x.dtype or \
            t.device != x.device:
        raise ValueError(f"{name} must have the shape, type and device of {of}")
    return _rows(t, name)[2]


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None,
               bias: torch.Tensor | None = None, eps: float = 1e-5, stats: bool = False,
               out: torch.Tensor | None = None, stream=None, ctx=None):
    """(y, mean, rstd) of layer norm over the last dimension
    (mx_layer_norm_fwd).  x: float32 or bfloat16, contiguous or 2-D with
    contiguous rows; weight, bias: float32.  mean and rstd (float32, one a row,
    for layer_norm_backward) are None unless `stats`."""
    dt = _check_type(x, "x")
    rows, cols, ldx = _rows(x, "x")
    dev = x.get_device()
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is not None:
            _check_like(t, name, dev, torch.float32, (cols,))
    if out is None:
        out = _empty_like(x, stream) if ldx == cols else _empty(x.shape, x.dtype, x, stream)
        ldy = cols
    else:
        ldy = _like_rows(out, "out", x, "x")
        _apart(out, "out", x, weight, bias)
    mean = rstd = None
    if stats:
        mean = _empty(rows, torch.float32, x, stream)
        rstd = _empty_like(mean, stream)
    rc = _lib.lib().mx_layer_norm_fwd(
        _handle(ctx, x), dt, x.data_ptr(), ldx, _ptr(weight), _ptr(bias), out.data_ptr(), ldy,
        _ptr(mean), _ptr(rstd), rows, cols, eps, _launch_stream(dev, stream))
    check(rc, "mx_layer_norm_fwd")
    return out, mean, rstd


def layer_norm_backward(grad_out: torch.Tensor, x: torch.Tensor, weight: torch.Tensor | None,
                        mean: torch.Tensor, rstd: torch.Tensor, dx: torch.Tensor | None = None,
                        dweight: torch.Tensor | None = None, dbias: torch.Tensor | None = None,
                        stream=None, ctx=None):
    """(dx, dweight, dbias) of layer_norm from its input and the mean and rstd
    that it gave (mx_layer_norm_bwd).  dweight and dbias are float32, summed
    over the rows in a fixed order."""
    dt = _check_type(x, "x")
    rows, cols, ldx = _rows(x, "x")
    dev, f32 = x.get_device(), torch.float32
    lddy = _like_rows(grad_out, "grad_out", x, "x")
    if weight is not None:
        _check_like(weight, "weight", dev, f32, (cols,))
    _check_like(mean, "mean", dev, f32, (rows,))
    _check_like(rstd, "rstd", dev, f32, (rows,))
    if dx is None:
        dx = _empty_like(x, stream) if ldx == cols else _empty(x.shape, x.dtype, x, stream)
        lddx = cols
    else:
        lddx = _like_rows(dx, "dx", x, "x")
        _apart(dx, "dx", grad_out, x, weight, mean, rstd, dweight, dbias)
    if dweight is None:
        dweight = _empty(cols, f32, x, stream) if weight is None else \
            _empty_like(weight, stream)
    else:
        _check_like(dweight, "dweight", dev, f32, (cols,))
        _apart(dweight, "dweight", grad_out, x, weight, mean, rstd, dbias)
    if dbias is None:
        dbias = _empty_like(dweight, stream)
    else:
        _check_like(dbias, "dbias", dev, f32, (cols,))
        _apart(dbias, "dbias", grad_out, x, weight, mean, rstd)
    h = _handle(ctx, x)
    L = _lib.lib()
    nb = L.mx_layer_norm_bwd_scratch_bytes(h, rows, cols)
    scratch = _empty(nb, torch.uint8, x, stream) if nb else None
    rc = L.mx_layer_norm_bwd(
        h, dt, grad_out.data_ptr(), lddy, x.data_ptr(), ldx, _ptr(weight), mean.data_ptr(),
        rstd.data_ptr(), dx.data_ptr(), lddx, dweight.data_ptr(), dbias.data_ptr(), rows, cols,
        _ptr(scratch), nb, _launch_stream(dev, stream))
    check(rc, "mx_layer_norm_bwd")
    return dx, dweight, dbias


def _gated_shape(x: torch.Tensor, w: torch.Tensor, transpose_w: bool, act: str):
    dt = _check_type(x, "x")
    if act not in _lib.ACTIVATIONS:
        raise ValueError(f"act must be one of {sorted(_lib.ACTIVATIONS)}, got {act!r}")
    dev = x.get_device()
    _check_like(x, "x", dev, x.dtype)
    _check_like(w, "w", dev, x.dtype)
    if x.dim() < 1 or w.dim() != 2:
        raise ValueError("x needs a last dimension, w two dimensions")
    K = x.shape[-1]
    M = x.numel() // K if K else math.prod(x.shape[:-1])
    two_f = w.shape[0] if transpose_w else w.shape[1]
    if two_f % 2 or w.shape[1 if transpose_w else 0] != K:
        raise ValueError(f"w has shape {tuple(w.shape)}, needs "
                         f"{('[2F, %d]' if transpose_w else '[%d, 2F]') % K}")
    if max(M, K, two_f) > _MAX_SIZE:
        raise ValueError(f"x and w have a dimension above {_MAX_SIZE}")
    return dt, dev, M, K, two_f // 2, x.shape[:-1]


def _pre_cols(F: int) -> int:
    """Columns of the saved pre-activations: both halves padded to 8."""
    return 2 * ((F + 7) // 8 * 8)


def gated_linear(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None = None,
                 act: str = "silu", transpose_w: bool = False, save: bool = False,
                 out: torch.Tensor | None = None, pre: torch.Tensor | None = None,
                 precision="default", stream=None, ctx=None):
    """(h, pre): h = act(g) * u with [g | u] = x op(w) + bias
    (mx_gated_linear_fwd).  x: [..., K] float32 or bfloat16; w: [K, 2F]
    (transpose_w=False) or [2F, K], the gate's half first; bias: [2F].  w, bias
    and h are of x's type.  pre, [g | u] in float32 for
    gated_linear_backward (each half padded to a multiple of 8 columns), is
    None unless `save` (or a buffer) is given."""
    dt, dev, M, K, F, lead = _gated_shape(x, w, transpose_w, act)
    if bias is not None:
        _check_like(bias, "bias", dev, x.dtype, (2 * F,))
    if out is None:
        out = _empty(lead + (F,), x.dtype, x, stream)
    else:
        _check_like(out, "out", dev, x.dtype, lead + (F,))
        _apart(out, "out", x, w, bias, pre)
    if pre is not None:
        _check_like(pre, "pre", dev, torch.float32, lead + (_pre_cols(F),))
        _apart(pre, "pre", x, w, bias)
    elif save:
        pre = _empty(lead + (_pre_cols(F),), torch.float32, x, stream)
    L, h, p = _lib.lib(), _handle(ctx, x), _prec(precision)
    nb = L.mx_gated_linear_workspace_bytes(h, dt, M, K, F, transpose_w, p, 0)
    ws = _empty(nb, torch.uint8, x, stream) if nb else None
    rc = L.mx_gated_linear_fwd(
        h, dt, x.data_ptr(), w.data_ptr(), _ptr(bias), out.data_ptr(), _ptr(pre), M, K, F,
        transpose_w, _lib.ACTIVATIONS[act], p, _ptr(ws), nb, _launch_stream(dev, stream))
    check(rc, "mx_gated_linear_fwd")
    return out, pre


def gated_linear_backward(grad_out: torch.Tensor, pre: torch.Tensor, x: torch.Tensor,
                          w: torch.Tensor, act: str = "silu", transpose_w: bool = False,
                          want_bias: bool = True, dx: torch.Tensor | None = None,
                          dw: torch.Tensor | None = None, dbias: torch.Tensor | None = None,
                          precision="default", stream=None, ctx=None):
    """(dx, dw, dbias) of gated_linear from the `pre` that it saved
    (mx_gated_linear_bwd); dbias is None without `want_bias`."""
    dt, dev, M, K, F, lead = _gated_shape(x, w, transpose_w, act)
    _check_like(grad_out, "grad_out", dev, x.dtype, lead + (F,))
    _check_like(pre, "pre", dev, torch.float32, lead + (_pre_cols(F),))
    if dx is None:
        dx = _empty_like(x, stream)
    else:
        _check_like(dx, "dx", dev, x.dtype, x.shape)
        _apart(dx, "dx", grad_out, pre, x, w, dw, dbias)
    if dw is None:
        dw = _empty_like(w, stream)
    else:
        _check_like(dw, "dw", dev, x.dtype, w.shape)
        _apart(dw, "dw", grad_out, pre, x, w, dbias)
    if dbias is not None:
        _check_like(dbias, "dbias", dev, x.dtype, (2 * F,))
        _apart(dbias, "dbias", grad_out, pre, x, w)
    elif want_bias:
        dbias = _empty(2 * F, x.dtype, x, stream)
    L, h, p = _lib.lib(), _handle(ctx, x), _prec(precision)
    nb = L.mx_gated_linear_workspace_bytes(h, dt, M, K, F, transpose_w, p, 1)
    ws = _empty(nb, torch.uint8, x, stream) if nb else None
    rc = L.mx_gated_linear_bwd(
        h, dt, grad_out.data_ptr(), pre.data_ptr(), x.data_ptr(), w.data_ptr(), dx.data_ptr(),
        dw.data_ptr(), _ptr(dbias), M, K, F, transpose_w, _lib.ACTIVATIONS[act], p, _ptr(ws), nb,
        _launch_stream(dev, stream))
    check(rc, "mx_gated_linear_bwd")
    return dx, dw, dbias


def adamw_state_values(codes: torch.Tensor, scale: torch.Tensor, out: torch.Tensor | None = None,
                       stream=None, ctx=None) -> torch.Tensor:
    """The moments that 8-bit AdamW states stand for, in bfloat16
    (mx_adamw_state_values): the first moment from int8 codes, the second from
    uint8 codes; scale holds one float32 for each 256 of them."""
    if not isinstance(codes, torch.Tensor) or not codes.is_cuda:
        raise TypeError("codes must be a CUDA tensor")
    if codes.dtype not in (torch.int8, torch.uint8):
        raise TypeError(f"codes must be int8 or uint8, got {codes.dtype}")
    dev, n = codes.get_device(), codes.numel()
    _check_like(codes, "codes", dev, codes.dtype)
    _check_like(scale, "scale", dev, torch.float32, (-(-n // 256),))
    if out is None:
        out = _empty(codes.shape, torch.bfloat16, codes, stream)
    else:
        _check_like(out, "out", dev, torch.bfloat16, codes.shape)
        _apart(out, "out", codes, scale)
    rc = _lib.lib().mx_adamw_state_values(
        _handle(ctx, codes), codes.data_ptr(), scale.data_ptr(), n, codes.dtype is torch.uint8,
        out.data_ptr(), _launch_stream(dev, stream))
    check(rc, "mx_adamw_state_values")
    return out


def status(device: int | None = None) -> tuple[int, int]:
    """(status, call site) of the device status word; synchronises, clears it."""
    return context_status(context(device))


def context_status(ctx) -> tuple[int, int]:
    """(status, call site) of one context's status word (mx_context_status):
    synchronises the context's device, clears the word."""
    where = ctypes.c_int32(0)
    rc = _lib.lib().mx_context_status(ctx, ctypes.byref(where))
    return rc, where.value


def reserve_workspace(nbytes: int, device: int | None = None) -> None:
    check(_lib.lib().mx_context_reserve_workspace(context(device), int(nbytes)),
          "mx_context_reserve_workspace")


def workspace_bytes(M: int, K: int, N: int, ta=False, tb=False, precision="default",
                    device: int | None = None) -> int:
    return int(_lib.lib().mx_matmul_workspace_bytes(context(device), M, K, N, int(ta), int(tb),
                                                    _prec(precision)))


def resolve_precision(M: int, K: int, N: int, precision="default",
                      device: int | None = None) -> str:
    p = _lib.lib().mx_matmul_resolve_precision(context(device), M, K, N, _prec(precision))
    return {v: k for k, v in PRECISIONS.items()}[p]
