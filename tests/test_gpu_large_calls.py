"""Calls of more workgroups than one dimension of a launch takes (2^24 of 256 threads).  They need most of the GPU's memory, and are
skipped where it is not free."""
from __future__ import annotations

import gc
import math

import pytest
import torch

from rsna_knee_efficiency_amd import optim

pytestmark = pytest.mark.gpu


@pytest.fixture
def free(dev):
    """Skips unless so many bytes are free; what the test made is given back behind it"""
    def need(n):
        gc.collect()
        torch.cuda.empty_cache()
        if torch.cuda.mem_get_info(dev)[0] < n + (4 << 30):
            pytest.skip(f"needs {n >> 30} GiB of free GPU memory")
    yield need
    gc.collect()
    torch.cuda.empty_cache()


def test_clipping_of_a_tensor_of_half_the_limit(dev, free):
    """2^37 elements: the last chunks are scaled too"""
    n = 1 << 37
    free(2 * n)
    x = torch.empty(n, dtype=torch.bfloat16, device=dev).zero_()
    at = [0, 8191, 8192, n // 2 + 1, n - 8193, n - 1]
    for i in at:
        x[i] = 1.0
    print("clip 2^37", flush=True)
    assert optim.clip_grad_norm([x], 0.5).item() == torch.tensor(math.sqrt(len(at))).item()
    want = torch.tensor(0.5 / math.sqrt(len(at))).bfloat16().item()
    assert [x[i].item() for i in at] == [want] * len(at) and not x[-3:-1].any() and not x[1:8191].any()
