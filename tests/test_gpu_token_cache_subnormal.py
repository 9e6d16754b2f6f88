"""Attention over blocks of subnormal bfloat16 values, against float64 with bfloat16's own smallest step as the only absolute term: an
output of zeros does not pass.  (Scales of such blocks are subnormal float32 numbers, codes times them exact multiples of 2^-149.)"""
from __future__ import annotations

import pytest
import torch

from rsna_knee_efficiency_amd.token_cache import QuantizedCache, cached_attention

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
INT8, E4M3 = torch.int8, torch.float8_e4m3fn
HALF = 2.0 ** -134                             # of bfloat16's smallest step


def _made(dev, codes, d, power, n, new, h, hk, mixed):
    g = torch.Generator(device=dev).manual_seed(new + d)
    q, k, v = (torch.randn((2, t, heads, d), generator=g, device=dev).to(BF16) for t, heads in ((new, h), (n, hk), (n, hk)))
    small = (v.double() * 2.0 ** power).to(BF16)
    block = torch.arange(n, device=dev) // 64
    where = (block % 5 == 2) & (block < n // 64)             # (the last block stays subnormal)
    v = torch.where(where[None, :, None, None], v, small) if mixed else small
    cache = QuantizedCache(2, n, hk, d, codes, BF16, dev)
    cache.append(k, v)
    return q, cache, where if mixed else torch.zeros_like(where)


SHAPES = [(2900, 2900, 16, 4), (2900, 700, 64, 2), (2900, 45, 4, 2), (900, 1, 8, 2)]


@pytest.mark.parametrize("n,new,h,hk", SHAPES)
@pytest.mark.parametrize("mixed", [False, True])
@pytest.mark.parametrize("codes,d", [(INT8, 64), (INT8, 128), (E4M3, 64), (E4M3, 128)])
@pytest.mark.parametrize("power", [-124, -130])
def test_a_token_that_sees_itself_alone(dev, power, codes, d, mixed, n, new, h, hk):
    """The value that the cache holds, rounded once: off by 2^-20 of it in float32 (weights in 16 bits are 2^8 exactly) and half a step"""
    print(f"itself 2^{power} {codes} {d} {mixed} new={new}", flush=True)
    q, cache, _ = _made(dev, codes, d, power, n, new, h, hk, mixed)
    got = cached_attention(q, cache, left=0).double()
    want = cache.read(dtype=F32)[1][:, n - new:].repeat_interleave(h // hk, 2).double()
    tol = want.abs() * (2.0 ** -8 + 2.0 ** -19) + HALF
    assert ((got - want).abs() <= tol).all()
    assert (want.abs() > tol).float().mean() > 0.3           # (an output of zeros is told apart)


@pytest.mark.parametrize("n,new,h,hk", SHAPES)
@pytest.mark.parametrize("mixed", [False, True])
@pytest.mark.parametrize("codes,d", [(INT8, 128), (E4M3, 64)])
@pytest.mark.parametrize("power", [-122, -126])
def test_a_few_tokens(dev, power, codes, d, mixed, n, new, h, hk):
    """Queries that see eight tokens, and beside ordinary blocks those among them that see subnormal ones alone.  Weights are rounded to
    8 bits at the coarsest and to 2^-29 of the largest, scores and sums are float32 (2^-16 of what they weigh), the result to bfloat16."""
    print(f"few 2^{power} {codes} {d} {mixed} new={new}", flush=True)
    q, cache, ordinary = _made(dev, codes, d, power, n, new, h, hk, mixed)
    got = cached_attention(q, cache, left=7).double()
    k, v = (x.double().repeat_interleave(h // hk, 2) for x in cache.read(dtype=F32))
    told = torch.zeros((), device=dev)
    for at in range(n - new, n, max(1, new // 150)):
        see = slice(max(0, at - 7), at + 1)
        p = torch.softmax((q[:, at - n + new, :, None].double() * k[:, see].transpose(1, 2)).sum(-1) / d ** 0.5, -1)[..., None]
        vv = v[:, see].transpose(1, 2)
        want, weighed = (p * vv).sum(2), (p * vv.abs()).sum(2)
        tol = weighed * (2.0 ** -8 + 2.0 ** -14) + 2.0 ** -29 * vv.abs().sum(2) + 2.0 ** -8 * want.abs() + HALF
        assert ((got[:, at - n + new] - want).abs() <= tol).all(), at
        if not ordinary[see].any():
            told = torch.maximum(told, (want.abs() > 2 * tol).float().mean())
    assert told > 0.3
