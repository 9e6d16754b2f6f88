"""Sizes at which the 8-bit cache's calls meet the GPU's own limits, on the host (CPU only, no kernel launches)."""
from __future__ import annotations

import ctypes

import pytest
import torch

from rsna_knee_efficiency_amd import hip, token_cache

P = 1 << 20                                    # a pointer that is not followed


def _workspace(B, S, T, H, HK, left, D=64):
    a = hip.CacheAttnArgs(hip.Cache(P, P, P, P, P, P, P, B, S, HK, D, 1, 0), q=P, out=P, T=T, H=H, left=left, scale=0.125)
    need = ctypes.c_uint64()
    hip.call("d8s_cache_attention_workspace", ctypes.byref(a), ctypes.byref(need))
    return need.value


def test_equal_shares_are_for_rows_that_a_launch_of_one_workgroup_each_takes():
    """Their join is a workgroup of 256 threads a row, and a launch has fewer than 2^32 threads: from 2^24 rows on the other form
    runs, which with as many key heads needs no workspace."""
    shares = _workspace(256, 2048, 1, 16 << 11, 1 << 11, 2048)
    assert shares > 0                          # 2^23 rows: in equal shares
    assert _workspace(256, 2048, 1, 16 << 12, 1 << 12, 2048) == 0            # 2^24 rows
    assert _workspace(255, 2048, 1, 16 << 12, 1 << 12, 2048) > 0


def _made(batch, capacity, key_heads):
    """A cache whose tensors lie on the host: what is refused before its device is looked at."""
    c = object.__new__(token_cache.QuantizedCache)
    c.__dict__.update(batch=batch, capacity=capacity, key_heads=key_heads, channels=64, codes=torch.int8, dtype=torch.bfloat16,
                      _lengths=torch.zeros(batch, dtype=torch.int32), device=torch.device("cuda:0"))
    return c


def _t(*shape):
    return torch.zeros((1,) * len(shape), dtype=torch.bfloat16).expand(shape)


@pytest.mark.parametrize("call", [
    lambda: token_cache.QuantizedCache(1 << 12, 10, 1 << 10, 64),
    lambda: _made(1 << 12, 1000, 2).append(_t(1 << 12, 1 << 20, 2, 64), _t(1 << 12, 1 << 20, 2, 64)),
    lambda: _made(2, 1000, 1).append(_t(2, (1 << 29) + 1, 1, 64), _t(2, (1 << 29) + 1, 1, 64)),
    lambda: token_cache.cached_attention(_t(2, 1 << 25, 2, 64), _made(2, 1000, 1)),
    lambda: token_cache.cached_attention(_t(2, (1 << 29) + 1, 1, 64), _made(2, 1000, 1)),
])
def test_sizes_that_are_too_large_are_wrong_values(call, monkeypatch):
    """As other wrong sizes are, and not failures of the library behind what the call has made already"""
    monkeypatch.setattr(token_cache, "_on_gpu", lambda *t: None)
    monkeypatch.setattr(token_cache, "_like", lambda *t: pytest.fail("an output was made"))
    with pytest.raises(ValueError, match="too many|too large|at most"):
        call()
