"""CPU tests of what the calls on layer norm, the gated layer and AdamW check
before a launch."""
from __future__ import annotations

import itertools

import pytest
import torch

from moonxi_net_b200 import ops


def _shares(out, t):
    try:
        ops._apart(out, "out", t)
    except ValueError as e:
        assert "share memory" in str(e)
        return True
    return False


def _elements(t):
    """The addresses of a tensor's elements, in units of one."""
    at = torch.tensor(0)
    for n, s in zip(t.shape, t.stride()):
        at = at[..., None] + torch.arange(n) * s
    return set((at + t.storage_offset()).flatten().tolist())


def test_outputs_that_share_memory_with_rows_in_between():
    """Refused if and only if an element is shared: every pair of row views of one
    buffer, of equal and of different pitches, and dense ones."""
    buf = torch.zeros(96)
    views = [buf[o:o + (r - 1) * p + c].as_strided((r, c), (p, 1), o)
             for o, r, c, p in itertools.product((0, 1, 3, 8, 13, 24), (1, 2, 4), (1, 3, 5, 8), (8, 11, 16))
             if o + (r - 1) * p + c <= 96]
    views += [buf[o:o + n] for o, n in ((0, 96), (0, 1), (95, 1), (20, 24), (7, 0))]
    places = [_elements(v) for v in views]
    assert len(views) > 150
    for (a, pa), (b, pb) in itertools.product(zip(views, places), repeat=2):
        assert _shares(a, b) == bool(pa & pb), (a.shape, a.stride(), a.storage_offset(),
                                                b.shape, b.stride(), b.storage_offset())


def test_outputs_of_other_types():
    buf = torch.zeros(64)
    half = buf.view(torch.bfloat16)
    assert _shares(half[10:20], buf[5:6]) and _shares(half[10:20], buf[9:12])
    assert not _shares(half[10:20], buf[10:12]) and not _shares(half[10:20], buf[:5])
    ops._apart(buf, "out", None, torch.zeros(4))
