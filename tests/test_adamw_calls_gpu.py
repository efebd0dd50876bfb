"""GPU tests of calls of nn.AdamW that would go wrong unseen."""
from __future__ import annotations

import pytest
import torch

from moonxi_net_b200 import nn

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def test_a_captured_step_needs_its_number_on_the_device(cuda_device):
    """Every replay would be the same step; nothing is counted for the refused call."""
    p, g = torch.ones(300, device="cuda"), torch.ones(300, device="cuda")
    opt = nn.AdamW([p])
    opt.step([g])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        graph.capture_begin()
        try:
            with pytest.raises(RuntimeError, match="device_step"):
                opt.step([g])
            _ = g + 1  # the capture goes on
        finally:
            graph.capture_end()
    torch.cuda.synchronize()
    assert opt.step_count == 1
    opt.step([g])
    assert opt.step_count == 2
