"""Sizes at which the 8-bit cache's calls meet the GPU's own limits, on the host (CPU only, no kernel launches)."""
from __future__ import annotations

import ctypes

from rsna_knee_efficiency_amd import hip

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
