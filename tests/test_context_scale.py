"""Attention's scale (CPU only): 1 / scale times a logarithm and scale times log2(e) must be float32 numbers, or every
gradient would be zero or no number."""
from __future__ import annotations

import ctypes

import pytest
import torch

from rsna_knee_efficiency_amd import context, hip

P = 1 << 20                                    # a pointer that is not followed


@pytest.mark.parametrize("scale", [1e-38, 1.5e-38, 7e-31, 1.5e30, 3e38])
def test_scales_out_of_range_are_refused(scale):
    a = hip.AttnArgs(**{n: P for n in ("q", "k", "v", "out", "lse", "dout", "dq", "dk", "dv", "workspace")},
                     ws_bytes=1 << 40, B=2, S=100, H=4, HK=2, D=64, dtype=1, left=10, right=0, sinks=2, scale=scale)
    t = hip.TokenArgs(**{n: P for n in ("q", "k", "v", "lengths", "out", "workspace")}, ws_bytes=1 << 40, B=2, S=1000,
                      H=4, HK=2, D=64, dtype=1, left=500, sinks=2, scale=scale)
    need = ctypes.c_uint64()
    for name, args in (("d8s_attention_workspace", a), ("d8s_attention_token_workspace", t)):
        with pytest.raises(hip.D8sError, match="scale"):
            hip.call(name, ctypes.byref(args), ctypes.byref(need))
        args.scale = 0.125
        hip.call(name, ctypes.byref(args), ctypes.byref(need))
    q, k = (torch.zeros((1, 4, 2, 64), dtype=torch.bfloat16) for _ in range(2))
    with pytest.raises(ValueError, match="scale"):
        context.window_attention(q, k, k, scale=scale)
    with pytest.raises(ValueError, match="one GPU"):       # (the first that these tensors are refused for)
        context.window_attention(q, k, k, scale=2.0 ** -100)
