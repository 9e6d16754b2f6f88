"""Calls of more workgroups than one dimension of a launch takes (2^24 of 256 threads).  They need most of the GPU's memory, and are
skipped where it is not free."""
from __future__ import annotations

import gc
import math

import pytest
import torch

from rsna_knee_efficiency_amd import optim
from rsna_knee_efficiency_amd.token_cache import QuantizedCache

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


def test_reading_all_of_a_large_cache(dev, free):
    """2^24 workgroups: a row that is full and one of 200 tokens"""
    n = 1 << 28
    free(n * 128 * 6)                          # (two rows of 64 channels: codes in 8 bits, and what is read in 16)
    cache = QuantizedCache(2, n, 1, 64, device=dev)
    x = torch.full((1, 1, 1, 64), 1.5, dtype=torch.bfloat16, device=dev).expand(2, n, 1, 64)
    cache.append(x, -x[:, :1].expand(2, n, 1, 64), torch.tensor([200, n], dtype=torch.int32, device=dev))
    print("read 2^28 tokens of two rows", flush=True)
    for got, want in zip(cache.read(), (1.5, -1.5)):
        assert (got[0, :200] == want).all() and not got[0, 200:1 << 20].any() and not got[0, 200::4097].any() and not got[0, -(1 << 20):].any()
        assert (got[1, :1 << 20] == want).all() and (got[1, ::4097] == want).all() and (got[1, -(1 << 20):] == want).all()
