"""The gradients' device memory stays in proportion to the GPU and to the inputs (CPU only: sizes, no launches)."""
from __future__ import annotations

import ctypes

import pytest

from rsna_knee_efficiency_amd import hip

P, KEYS, SLOTS = 1 << 20, 128, 256 * 3         # a pointer that is not followed; keys a workgroup; workgroups the GPU holds


@pytest.mark.parametrize("b,s,h,hk,d,left,right,sinks", [
    (1, 22528, 32, 8, 128, 255, 0, 4096), (1, 65536, 16, 4, 128, 0, 0, 65536), (4, 8192, 8, 8, 64, 100, 100, 8192),
    (1, 1 << 20, 8, 1, 64, 63, 0, 1 << 16), (2, 8199, 16, 4, 128, 1023, 0, 4), (1, 300, 64, 1, 64, 10, 10, 40)])
@pytest.mark.parametrize("dtype", [1, 2])
def test_parts_of_many_first_tokens(b, s, h, hk, d, left, right, sinks, dtype):
    """One float32 dk and dv of 128 keys for two workgroups a slot of the GPU, and for two to every run of 128 keys, beside
    a few numbers a query."""
    a = hip.AttnArgs(**{n: P for n in ("q", "k", "v", "out", "lse", "dout", "dq", "dk", "dv", "workspace")},
                     ws_bytes=1 << 40, B=b, S=s, H=h, HK=hk, D=d, dtype=dtype, left=left, right=right, sinks=sinks, scale=0.125)
    need = ctypes.c_uint64()
    hip.call("d8s_attention_workspace", ctypes.byref(a), ctypes.byref(need))
    runs = b * hk * -(-s // KEYS)
    assert need.value <= (2 * SLOTS + 2 * runs) * 2 * KEYS * d * 4 + 8 * b * (h + hk) * s + 1024
