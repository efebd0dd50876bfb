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


def test_copies_that_moved_are_refused(cuda_device):
    """A bfloat16 copy that was given other memory would go stale while the old
    memory is written."""
    p, g = torch.ones(300, device="cuda"), torch.ones(300, device="cuda")
    c = torch.zeros(300, device="cuda", dtype=BF16)
    old = c.detach()
    opt = nn.AdamW([p, p.clone()], copies=[None, c])
    opt.step([g, g])
    before = old.clone(), p.clone()
    c.data = torch.zeros(300, device="cuda", dtype=BF16)
    with pytest.raises(ValueError, match="copies\\[1\\] was given other memory"):
        opt.step([g, g])
    assert torch.equal(old, before[0]) and torch.equal(p, before[1]) and opt.step_count == 1
