"""Powers of two moved between queries, keys and the scale change nothing of attention over the 8-bit cache, as long as each is in its
type's range: the scores are the same numbers, and so is every bit of the result."""
from __future__ import annotations

import pytest
import torch

from rsna_knee_efficiency_amd.token_cache import QuantizedCache, cached_attention

pytestmark = pytest.mark.gpu

BF16, INT8, E4M3 = torch.bfloat16, torch.int8, torch.float8_e4m3fn


@pytest.mark.parametrize("new,h,hk", [(1, 8, 2), (45, 4, 2), (700, 64, 2)])
@pytest.mark.parametrize("codes,d", [(INT8, 64), (E4M3, 128)])
@pytest.mark.parametrize("up,keys", [(120, -33), (126, -60), (95, 0), (-100, 60), (-120, 24), (-133, 38), (-133, 50), (60, -100)])
def test_powers_of_two(dev, up, keys, codes, d, new, h, hk):
    """Queries times 2^up, keys times 2^keys, the scale times what undoes both.  (Subnormal queries over full blocks alone: in the last
    block they are the matrix unit's own operands, and it rounds sums of their products otherwise in the last place.)"""
    print(f"2^{up} 2^{keys} {codes} {d} new={new}", flush=True)
    g, n = torch.Generator(device=dev).manual_seed(new + d), 2944 if up < -126 else 3000
    # whole numbers up to 3: queries of 2^-133 and three times that are in the type
    q = torch.randint(-3, 4, (1, new, h, d), generator=g, device=dev).double()
    k, v = (torch.randn((1, n, hk, d), generator=g, device=dev).to(BF16) for _ in range(2))
    k = torch.where(k.abs() < 2.0 ** -12, 0.0, k)            # (so that no key leaves the type's normal numbers)

    def out(up, keys, scale):
        cache = QuantizedCache(1, n, hk, d, codes, BF16, dev)
        cache.append((k.double() * 2.0 ** keys).to(BF16), v)
        x = (q * 2.0 ** up).to(BF16)
        assert torch.equal(x.double(), q * 2.0 ** up)
        return cached_attention(x, cache, scale=scale)
    scale = 4.0 if up < -126 else 0.0625       # (so that the scale times that of the keys passes 2^128)
    assert 2.0 ** -100 <= scale * 2.0 ** -(up + keys) <= 2.0 ** 100
    want = out(0, 0, scale)
    assert want.isfinite().all() and torch.equal(out(up, keys, scale * 2.0 ** -(up + keys)), want)
