"""CPU tests of layer norm, the gated linear layer and AdamW: what they refuse
before anything reaches a device, and their size queries without one."""
from __future__ import annotations

import ctypes

import pytest
import torch

from moonxi_net_b200 import _lib, nn, ops


def test_tensors_off_the_gpu_are_refused():
    x, w = torch.zeros(4, 8), torch.zeros(8, 12)
    with pytest.raises(TypeError, match="x must be a CUDA tensor"):
        ops.layer_norm(x)
    with pytest.raises(TypeError, match="x must be a CUDA tensor"):
        ops.layer_norm_backward(x, x, None, torch.zeros(4), torch.zeros(4))
    with pytest.raises(TypeError, match="x must be a CUDA tensor"):
        ops.gated_linear(x, w)
    with pytest.raises(TypeError, match="x must be a CUDA tensor"):
        ops.gated_linear_backward(torch.zeros(4, 6), torch.zeros(4, 16), x, w)
    with pytest.raises(TypeError, match="codes must be a CUDA tensor"):
        ops.adamw_state_values(torch.zeros(4, dtype=torch.int8), torch.zeros(1))
    with pytest.raises(TypeError, match="must be a CUDA tensor"):
        nn.AdamW([x])
    with pytest.raises(TypeError, match="must be a CUDA tensor"):
        ops.layer_norm(None)


def test_optimizer_arguments_are_checked_first():
    with pytest.raises(ValueError, match="at least one tensor"):
        nn.AdamW([])
    with pytest.raises(ValueError, match="state_bits"):
        nn.AdamW([torch.zeros(4)], state_bits=16)


def test_row_views():
    """Rows of the last dimension: contiguous, or 2-D with a row stride."""
    assert ops._rows(torch.zeros(3, 5, 8), "t") == (15, 8, 8)
    assert ops._rows(torch.zeros(8), "t") == (1, 8, 8)
    assert ops._rows(torch.zeros(6, 20)[:, 3:11], "t") == (6, 8, 20)
    assert ops._rows(torch.zeros(0, 8), "t") == (0, 8, 8)
    for bad in (torch.zeros(8, 6).t(), torch.zeros(2, 6, 20)[:, :, :8], torch.zeros(3, 0),
                torch.zeros(1, 8).expand(4, 8), torch.tensor(1.0)):
        with pytest.raises(ValueError):
            ops._rows(bad, "t")


def test_saved_pre_activations_are_padded_to_eight():
    assert [ops._pre_cols(f) for f in (1, 8, 9, 1000, 2731)] == [16, 16, 32, 2000, 5472]


def test_scratch_grows_with_launches_only_when_clipping():
    L = _lib.lib()
    assert L.mx_adamw_scratch_bytes(1, 0) == L.mx_adamw_scratch_bytes(10000, 0) >= 16
    one, many = L.mx_adamw_scratch_bytes(320, 1), L.mx_adamw_scratch_bytes(321, 1)
    assert many > one > L.mx_adamw_scratch_bytes(320, 0)


def test_calls_without_device_report_status():
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    L = _lib.lib()
    buf = (ctypes.c_float * 64)()
    p = ctypes.addressof(buf)
    assert L.mx_layer_norm_fwd(None, 0, p, 4, None, None, p, 4, None, None, 1, 4, 1e-5, None) == \
        _lib.MX_ERR_NO_DEVICE
    assert L.mx_layer_norm_bwd(None, 0, p, 4, p, 4, None, p, p, p, 4, p, p, 1, 4, p, 256, None) == \
        _lib.MX_ERR_NO_DEVICE
    assert L.mx_layer_norm_bwd_scratch_bytes(None, 4, 4) == 0
    assert L.mx_gated_linear_fwd(None, 0, p, p, None, p, None, 1, 1, 1, 0, 0, 0, None, 0, None) == \
        _lib.MX_ERR_NO_DEVICE
    assert L.mx_gated_linear_bwd(None, 0, p, p, p, p, p, p, None, 1, 1, 1, 0, 0, 0, None, 0, None) \
        == _lib.MX_ERR_NO_DEVICE
    assert L.mx_gated_linear_workspace_bytes(None, 1, 8, 8, 8, 0, 0, 1) == 0
    t = (_lib.AdamWTensor * 1)()
    assert L.mx_adamw_step(None, t, 1, 32, 1e-3, 0.9, 0.99, 1e-8, 1, None, 0.0, None, None, 0,
                           None) == _lib.MX_ERR_NO_DEVICE
    assert L.mx_adamw_state_values(None, p, p, 4, 0, p, None) == _lib.MX_ERR_NO_DEVICE
