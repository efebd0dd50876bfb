"""More GPU tests of the gated linear layer, with the checks and tolerances of
test_gated_gpu.py."""
from __future__ import annotations

import pytest
import torch

from test_gated_gpu import _run_and_check

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
