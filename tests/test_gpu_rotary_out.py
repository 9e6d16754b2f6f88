"""Rotary positions written into x's own memory at other places than x's."""
from __future__ import annotations

import pytest
import torch

from rsna_knee_efficiency_amd import context

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_out_across_x(dev, dtype):
    """One token on, one token back, some heads on, beside: as into memory of its own."""
    g = torch.Generator(device=dev).manual_seed(1)
    buf = torch.randn((2, 3001, 12, 64), generator=g, device=dev).to(dtype)
    pos = torch.randint(0, 90, (3000, 3), generator=g, device=dev, dtype=torch.int32)
    for put, get in (((slice(1, 3001), slice(0, 12)), (slice(0, 3000), slice(0, 12))),
                     ((slice(0, 3000), slice(0, 12)), (slice(1, 3001), slice(0, 12))),
                     ((slice(0, 3000), slice(2, 10)), (slice(0, 3000), slice(0, 8))),
                     ((slice(0, 3000), slice(6, 12)), (slice(0, 3000), slice(0, 6)))):
        memory = buf.clone()
        x, out = memory[:, get[0], get[1]], memory[:, put[0], put[1]]
        want = context.rotary(x, pos, (8, 12, 12))
        untouched = memory.clone()
        untouched[:, put[0], put[1]] = 0
        assert context.rotary(x, pos, (8, 12, 12), out=out) is out
        assert torch.equal(out, want)
        memory[:, put[0], put[1]] = 0
        assert torch.equal(memory, untouched)
