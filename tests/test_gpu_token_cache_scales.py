"""Attention over the 8-bit cache where blocks' values differ by more than float32's sums can hold together, row by row against float64
by what each row sees.

A row's bound: weights are rounded to float16 between the products, 2^-11 of each; a float16 number's last place is 2^-24, and a weight is
2^8 times its value over the row's largest, times a power of two of 1/16 at least, so a weight that float16 does not hold is off by
2^-29 of the largest, and by no more than itself; the last block's weights are rounded to the inputs' type.  Scores and sums are float32.
A row that sees values of 2^63 or more may hold its sums in units of 2^64: their last place is then 2^-149 times that, over the
2^8 of the largest weight."""
from __future__ import annotations

import math

import pytest
import torch

from rsna_knee_efficiency_amd.token_cache import QuantizedCache, cached_attention

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
INT8, E4M3 = torch.int8, torch.float8_e4m3fn


def _oracle(q, k, v, left, right, sinks, scale):
    """(out, bound) of one row's last tokens: q (tokens, heads, channels), k and v (length, key heads, channels) in float32, by key head"""
    t, h, d = q.shape
    n, hk = k.shape[:2]
    i, j = torch.arange(n - t, n, device=q.device)[:, None], torch.arange(n, device=q.device)[None]
    see = (j <= i + (n if right is None else right)) & ((j >= i - (n if left is None else left)) | (j < sinks))
    sums = n / 16 + 160                        # float32 sums over a block's tokens and over the blocks
    u = torch.finfo(q.dtype).eps / 2
    tail = n // 64 * 64
    out, tol = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for head in range(h):
        x, kk, vv = q[:, head].double(), k[:, head // (h // hk)].double(), v[:, head // (h // hk)].double()
        s = (x @ kk.T * scale).masked_fill(~see, -math.inf)
        es = 2 * d * 2.0 ** -24 * (x.abs() @ kk.abs().T).amax() * scale + 2.0 ** -18
        p = torch.softmax(s, -1).nan_to_num(0.0)
        o, av = p @ vv, vv.abs()
        high = (see & (av.amax(1) >= 2.0 ** 63)).any(1, keepdim=True)
        e = (2.0 ** -11 + 4 * es + sums * 2.0 ** -24) * (p @ av) + max(0.0, u - 2.0 ** -11) * (p[:, tail:] @ av[tail:])
        e = e + (2 * p).clamp(max=2.0 ** -29) @ av + u * o.abs() + torch.finfo(q.dtype).smallest_normal * u
        out[:, head], tol[:, head] = o, e + sums * 2.0 ** -149 * torch.where(high, 2.0 ** 56, 2.0 ** -8)
    return out, tol


def _check(cache, q, left=None, right=0, sinks=0, scale=None):
    got = cached_attention(q, cache, left, right, sinks, scale=scale)
    assert torch.equal(got, cached_attention(q, cache, left, right, sinks, scale=scale))
    k, v = cache.read(dtype=F32)
    for r, n in enumerate(cache.lengths.tolist()):
        want, tol = _oracle(q[r], k[r, :n], v[r, :n], left, right, sinks, scale or 1 / math.sqrt(q.shape[-1]))
        off = (got[r].double() - want).abs()
        bad = ~(off <= tol)
        assert not bad.any(), (r, bad.sum().item(), *(x[bad][0].item() for x in (got[r], want, tol)))
    return got


# (block -> the power of two of its values' largest)
SIZES = {
    "a large block": lambda b, n: torch.where(b == n // 3, 128.0, 0.0),
    "a large block, the others small": lambda b, n: torch.where(b == n // 3, 128.0, -66.0),
    "falling": lambda b, n: torch.tensor([128.0, 0.0, -20.0, -66.0], device=b.device)[b * 4 // n],
    "rising": lambda b, n: torch.tensor([-66.0, -20.0, 0.0, 128.0], device=b.device)[b * 4 // n],
    "in turn": lambda b, n: torch.tensor([128.0, 0.0, -20.0, -66.0], device=b.device)[b % 4],
    "2^100 and 2^-20": lambda b, n: torch.where(b % 9 == 4, 100.0, -20.0),
    "2^50 and 2^-50": lambda b, n: torch.where(b % 3 == 1, 50.0, -50.0),
    "2^30 and 2^-28": lambda b, n: torch.where(b % 5 == 1, 30.0, -28.0),
}
# batch, new, heads, key heads, window: many rows a key head (128 or 256 a workgroup), a share of blocks each and joined, a few
SHAPES = [(1, 2500, 16, 4, 300), (1, 2500, 16, 4, None), (1, 700, 64, 2, None), (1, 45, 4, 2, 300), (3, 1, 8, 2, 1500)]


@pytest.mark.parametrize("batch,new,h,hk,left", SHAPES)
@pytest.mark.parametrize("codes,d", [(INT8, 64), (INT8, 128), (E4M3, 64), (E4M3, 128)])
def test_values_that_a_row_does_not_see(dev, codes, d, batch, new, h, hk, left):
    """Blocks of up to bfloat16's largest value beside others, in every order: a row's result is that of the blocks it sees."""
    g, n = torch.Generator(device=dev).manual_seed(new + d), 3000 if new > 1 else 2990
    q, k = (torch.randn((batch, t, heads, d), generator=g, device=dev).to(BF16) for t, heads in ((new, h), (n, hk)))
    unit = torch.rand((batch, n, hk, d), generator=g, device=dev).double() * 2 - 1
    block = torch.arange(n, device=dev) // 64
    for name, power in SIZES.items():
        print(f"{name} {codes} {d} new={new} left={left}", flush=True)
        v = (unit * 0.99 * torch.exp2(power(block, n // 64 + 1).double())[None, :, None, None]).to(BF16)
        assert v.isfinite().all()
        cache = QuantizedCache(batch, n, hk, d, codes, BF16, dev)
        cache.append(k, v)
        _check(cache, q, left)
        _check(cache, q, left, 70, 5)


@pytest.mark.parametrize("new,h,hk", [(2500, 16, 4), (700, 64, 2), (45, 4, 2), (1, 8, 2)])
@pytest.mark.parametrize("codes", [INT8, E4M3])
def test_values_whose_weights_are_zero(dev, codes, new, h, hk):
    """Large blocks that a row sees, with scores so far below the others that their weights are zero; and a head's channels that
    are zero in them."""
    g, n, d = torch.Generator(device=dev).manual_seed(new), 3000, 64
    q, k = (torch.randn((1, t, heads, d), generator=g, device=dev) for t, heads in ((new, h), (n, hk)))
    unit = torch.rand((1, n, hk, d), generator=g, device=dev).double() * 2 - 1
    block = torch.arange(n, device=dev) // 64
    for name, large in (("once", block == 11), ("often", block % 5 == 2), ("at first", block < 20)):
        for power, small in ((120.0, 0.0), (128.0, -60.0), (100.0, -20.0), (30.0, -30.0)):
            print(f"zero weights: {name} 2^{power} 2^{small} {codes} new={new}", flush=True)
            v = unit * 0.99 * torch.exp2(torch.where(large, power, small).double())[None, :, None, None]
            low = torch.where(large[None, :, None, None], k - 40, k)
            cache = QuantizedCache(1, n, hk, d, codes, BF16, dev)
            cache.append(low.to(BF16), v.to(BF16))
            _check(cache, (q * 0.2 + 2).to(BF16))
            v[:, large, :, ::3] = 0
            cache = QuantizedCache(1, n, hk, d, codes, BF16, dev)
            cache.append(k.to(BF16), v.to(BF16))
            _check(cache, q.to(BF16))


@pytest.mark.parametrize("batch,new,h,hk", [(1, 2500, 16, 4), (1, 700, 64, 2), (1, 45, 4, 2), (3, 2, 8, 2)])
@pytest.mark.parametrize("codes,d", [(INT8, 128), (E4M3, 64)])
def test_tokens_of_the_last_block_that_a_row_does_not_see(dev, codes, d, batch, new, h, hk):
    """Large values of single tokens of the last block, the others far below: queries before such a token keep all of theirs."""
    g, n = torch.Generator(device=dev).manual_seed(new), 3000           # 56 tokens in the last block
    q, k = (torch.randn((batch, t, heads, d), generator=g, device=dev).to(BF16) for t, heads in ((new, h), (n, hk)))
    unit = torch.rand((batch, n, hk, d), generator=g, device=dev).double() * 2 - 1
    for at in ([n - 1], [n - 20], [n - 56], [n - 50, n - 9]):
        for small in (0.0, -66.0, -100.0):
            print(f"last block {at} 2^{small} {codes} new={new}", flush=True)
            v = unit * 2.0 ** small
            v[:, at, 0, 5] = 2.0 ** 127
            v[:, at, hk - 1, d - 1] = -(2.0 ** 64)
            cache = QuantizedCache(batch, n + 40, hk, d, codes, BF16, dev)
            cache.append(k, v.to(BF16))
            _check(cache, q)
            _check(cache, q, 40, 3, 2)


@pytest.mark.parametrize("codes,d", [(INT8, 128), (E4M3, 64)])
@pytest.mark.parametrize("new,h,hk", [(2500, 16, 4), (700, 64, 2), (45, 4, 2)])
def test_ragged_requests_over_blocks_far_apart(dev, codes, d, new, h, hk):
    """Requests of every length with some of the new tokens, among blocks of 2^120 and 2^-20 and one that is not a number: queries that
    see nothing of it have their own results, those that see its value's block have none, what lies past a count is zeros and not read."""
    g, n, left = torch.Generator(device=dev).manual_seed(new), 3000, 300
    lengths, counts = [3000, 2000, 64, 0, 1700], [new, new // 3, 64, 5, 0]
    b = len(lengths)
    q, k = (torch.randn((b, t, heads, d), generator=g, device=dev).to(BF16) for t, heads in ((new, h), (n, hk)))
    block = torch.arange(n, device=dev) // 64
    v = (torch.rand((b, n, hk, d), generator=g, device=dev).double() * 2 - 1) * torch.exp2(torch.where(block % 4 == 1, 120.0, -20.0).double())[None, :, None, None]
    v = v.to(BF16)
    v[:, 64 * 25 + 7, 0, 3] = float("nan")
    cache = QuantizedCache(b, n, hk, d, codes, BF16, dev)
    cache.append(k, v, torch.tensor(lengths, dtype=torch.int32, device=dev))
    for r, c in enumerate(counts):
        q[r, c:] = float("nan")
    print(f"ragged {codes} {d} new={new}", flush=True)
    got = cached_attention(q, cache, left, 0, counts=torch.tensor(counts, dtype=torch.int32, device=dev))
    kk, vv = cache.read(dtype=F32)
    for r, (m, c) in enumerate(zip(lengths, counts)):
        c = min(c, new)
        assert not got[r, c:].any()
        s = min(c, m)
        if not s:
            assert not got[r].any()
            continue
        at = torch.arange(m - s, m, device=dev)
        sees = (at >= 64 * 25) & (at - left < 64 * 26) & (m >= 64 * 26)
        want, tol = _oracle(q[r, c - s:c], kk[r, :m], vv[r, :m].nan_to_num(0.0), left, 0, 0, d ** -0.5)
        mine, per = got[r, c - s:c], h // hk
        bad = torch.zeros((s, h), dtype=torch.bool, device=dev)
        bad[:, :per] = sees[:, None]
        assert mine[bad].isnan().all()
        assert ((mine.double() - want).abs() <= tol)[~bad].all()
        if c > s:
            assert not got[r, :c - s].any()
