"""More GPU tests of nn.AdamW's 8-bit moments."""
from __future__ import annotations

import pytest
import torch

from moonxi_net_b200 import nn

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def test_blocks_without_a_gradient_keep_zeros(cuda_device):
    """Zero has code 0 in a block whose moments are all zero, and a value that is
    zero there stays zero, and its copy too."""
    n = 256 * 3 + 100
    p = torch.zeros(n, device="cuda")
    copy = torch.ones(n, device="cuda", dtype=BF16)
    opt = nn.AdamW([p], state_bits=8, lr=0.1, betas=(0.9, 0.95), copies=[copy])
    g = torch.zeros(n, device="cuda")
    g[256:300] = 0.01  # one block has gradients
    alone = torch.cat((torch.arange(256), torch.arange(512, n))).cuda()
    for _ in range(4):
        opt.step([g])
        mq, ms, vq, vs = opt.state[0]
        assert (mq[alone] == 0).all() and (vq[alone] == 0).all()
        assert (p[alone] == 0).all() and (copy[alone] == 0).all()
    assert (mq[256:300] > 0).all() and (vq[256:300] > 0).all() and (p[256:300] < 0).all()


@pytest.mark.parametrize("exponent", [-118, -116, -114, -112, -110, -60])
def test_blocks_of_tiny_moments(cuda_device, exponent):
    """Codes do not depend on the size of the block's largest moment.  The step
    computes m in float32 (gradients are powers of two times a root of the code:
    m = 0.5 g to half a unit in the last place), the code is the nearest one in
    the root, or floor(root + 1/64) below 0.5 / (1 - sqrt(0.5)) + 1; the root's own
    roundings are 2^-10 of a code."""
    k = torch.arange(256, device="cuda") % 128
    g = (k.double() / 127).square() * 2.0 ** exponent * 2
    sign = torch.where(torch.arange(256, device="cuda") < 128, 1.0, -1.0)
    p = torch.zeros(256, device="cuda")
    opt = nn.AdamW([p], state_bits=8, lr=0.1, betas=(0.5, 0.9))
    opt.step([(g * sign).float()])
    mq, ms = opt.state[0][:2]
    assert abs(float(ms) / 2.0 ** exponent - 1) <= 2.0 ** -22
    assert torch.equal(mq.int(), (k * sign).int())
    assert opt.state[0][3].isfinite().all()
