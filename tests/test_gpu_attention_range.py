"""Attention's gradients in float16 over the range of gradients that training gives: a loss averaged over thousands of
tokens, a loss scaled up, a few rows far larger than the others.

The oracle is the formula in float64, and errors are compared by their norm.  With u = 2^-11 (a float16 rounding is off
by at most u of the value, its own last step 2^-25 below 2^-14), every rounded value is off by its own independent
error, so the norm of a sum of n of them is at most u times the root of the sum of the terms' squares (their root mean
square is below 0.6 u).  What is rounded: dS (or P, for dv) before the product, out before rowsum(do out), the result;
P has an error of es beside, from its score in float32."""
from __future__ import annotations

import math

import pytest
import torch

from rsna_knee_efficiency_amd import context

pytestmark = pytest.mark.gpu

U, STEP = 2.0 ** -11, 2.0 ** -25


def _heads(t, per=1):
    return t.double().transpose(1, 2).repeat_interleave(per, 1)


def _oracle(q, k, v, dout, see, scale):
    """(dq, dk, dv) in float64 as (batch, heads, tokens, channels) and the norms their errors stay below"""
    b, n, h, d = q.shape
    per = h // k.shape[2]
    q, k, v, do = _heads(q), _heads(k, per), _heads(v, per), _heads(dout)
    s = (q @ k.transpose(2, 3) * scale).masked_fill(~see, -math.inf)
    es = 2 * d * 2.0 ** -24 * (q.norm(dim=-1).amax() * k.norm(dim=-1).amax()) * scale + 2.0 ** -19
    p = torch.where(see, torch.softmax(s, -1), 0.0)          # (a row that sees nothing: zeros)
    o = p @ v
    row = (do * o).sum(-1, keepdim=True)
    ds = p * (do @ v.transpose(2, 3) - row)
    u = U + 2 * es
    # out's own rounding, and that of the P it came from
    erow = ((do * o).square().sum(-1, keepdim=True) + (do.square() * (p.square() @ v.square())).sum(-1, keepdim=True)).sqrt() * u

    def shared(t):
        return t.reshape(b, -1, per, *t.shape[2:]).sum(2)
    dq, dk, dv = ds @ k * scale, shared(ds.transpose(2, 3) @ q) * scale, shared(p.transpose(2, 3) @ do)

    def bound(want, left, right, by):
        terms = (left.square() @ right.square()).sum().sqrt() * by
        return U * want.norm() + STEP * math.sqrt(want.numel()) + u * terms
    edq = bound(dq, ds, k, scale) + ((p @ k) * erow).norm() * scale
    edk = bound(dk, ds.transpose(2, 3), q, scale) + ((p.transpose(2, 3) @ (erow * q)).norm()) * scale
    edv = bound(dv, p.transpose(2, 3), do, 1.0)
    return (dq, dk, dv), (edq, edk, edv)


def _check(q, k, v, dout, scale=None, mask=None, **how):
    n = q.shape[1]
    how = dict(left=None, right=None, sinks=0) | how
    i, j = torch.arange(n, device=q.device)[:, None], torch.arange(n, device=q.device)[None]
    left, right = (n if how[side] is None else how[side] for side in ("left", "right"))
    see = (j <= i + right) & ((j >= i - left) | (j < how["sinks"]))
    see = see[None, None] if mask is None else see[None, None] & mask[:, None, None]
    out, lse = context.window_attention_forward(q, k, v, **how, key_mask=mask, scale=scale)
    got = context.window_attention_backward(dout, q, k, v, out, lse, **how, key_mask=mask, scale=scale)
    want, tol = _oracle(q, k, v, dout, see, 1 / math.sqrt(q.shape[-1]) if scale is None else scale)
    for name, x, y, e in zip(("dq", "dk", "dv"), got, want, tol):
        off = (x.double().transpose(1, 2) - y).norm()
        print(f"{name}: off by {(off / y.norm()).item():.2e}, bound {(e / y.norm()).item():.2e} of its norm", flush=True)
        assert off <= e, name
    return got


def _inputs(dev, seed, b, n, h, hk, d, size, qs=1.5, vs=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    shapes = ((b, n, h, d), (b, n, hk, d), (b, n, hk, d), (b, n, h, d))
    return [(torch.randn(s, generator=g, device=dev) * x).half() for s, x in zip(shapes, (qs, 1.0, vs, size))]


@pytest.mark.parametrize("size", [1.0, 1e-3, 1e-4, 1e-5])
@pytest.mark.parametrize("d,h,hk", [(64, 1, 1), (128, 2, 1)])
def test_gradients_of_an_averaged_loss(dev, size, d, h, hk):
    """Thousands of visible keys: dS is a thousandth of a gradient that is small by itself."""
    _check(*_inputs(dev, 1, 1, 3000, h, hk, d, size))
    _check(*_inputs(dev, 2, 1, 3001, h, hk, d, size), left=1000, right=0, sinks=5)


@pytest.mark.parametrize("d", [64, 128])
def test_gradients_of_a_scaled_loss(dev, d):
    """dP beyond float16's largest value, results within it."""
    q, k, v, do = _inputs(dev, 3, 2, 16, 2, 1, d, 1e4, qs=4.0, vs=8.0)
    got = _check(q, k, v, do, scale=2.0 ** -7)
    assert all(t.isfinite().all() for t in got)


def test_rows_of_all_sizes(dev):
    """Summary tokens whose gradient is ten thousand times the others', and rows whose gradient is zero."""
    q, k, v, do = _inputs(dev, 4, 1, 2000, 2, 2, 64, 1e-4)
    do[:, :4] *= 1e4
    do[:, 500:700] = 0
    _check(q, k, v, do, left=600, right=600, sinks=4)
    _check(q, k, v, torch.zeros_like(do), left=600, right=600, sinks=4)


def test_unseen_rows_cost_nothing(dev):
    """What a masked key holds, and the gradient of a query that sees nothing, cost the others no bits."""
    q, k, v, do = _inputs(dev, 5, 1, 700, 2, 1, 64, 1e-4)
    mask = torch.ones((1, 700), dtype=torch.bool, device=dev)
    mask[:, 100:300] = False
    how = dict(left=20, right=20, sinks=0)
    want = _check(q, k, v, do, mask=mask, **how)
    far_do = do.clone()
    far_do[:, 120:280] = 6e4                   # these see masked keys only
    for x in (6e4, float("inf"), float("nan")):
        far_v = v.clone()
        far_v[:, 100:300] = x
        out, lse = context.window_attention_forward(q, k, far_v, **how, key_mask=mask)
        got = context.window_attention_backward(far_do, q, k, far_v, out, lse, **how, key_mask=mask)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), x


@pytest.mark.parametrize("dtype,d", [(torch.float16, 64), (torch.float16, 128), (torch.bfloat16, 64), (torch.bfloat16, 128)])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_unseen_rows_are_not_used(dev, dtype, d, bad):
    """Queries that see nothing, and their gradient, may hold anything: no other row's gradient changes, theirs are zeros."""
    q, k, v, do = (t.to(dtype) for t in _inputs(dev, 6, 2, 500, 4, 2, d, 1.0))
    mask = torch.ones((2, 500), dtype=torch.bool, device=dev)
    mask[:, 100:300] = False
    mask[1, 310:] = False
    for left, right, sinks in ((20, 20, 0), (5, 0, 0)):
        how = dict(left=left, right=right, sinks=sinks, key_mask=mask)
        out, lse = context.window_attention_forward(q, k, v, **how)
        want = context.window_attention_backward(do, q, k, v, out, lse, **how)
        assert all(t.isfinite().all() for t in want)
        unseen = (lse == -math.inf)[:, 0]
        assert unseen[:, 130:270].all() and unseen[1, 340:].all()
        for both in ((True, False), (False, True), (True, True)):
            far = [t.clone() for t in (q, do)]
            for t, on in zip(far, both):
                t[unseen] = bad if on else t[unseen]
            again = context.window_attention_forward(far[0], k, v, **how)
            assert torch.equal(again[0], out) and torch.equal(again[1], lse)
            got = context.window_attention_backward(far[1], far[0], k, v, out, lse, **how)
            assert all(torch.equal(a, b) for a, b in zip(got, want)) and not got[0][unseen].any()


def test_many_first_tokens(dev):
    """More tiles of first tokens than the GPU needs workgroups: their gradients are split into few shares."""
    q, k, v, do = _inputs(dev, 7, 1, 4000, 16, 8, 64, 1e-3)
    _check(q, k, v, do, left=3, right=0, sinks=4000)
    _check(q, k, v, do, left=100, right=0, sinks=1500)


@pytest.mark.parametrize("high", [17.4, 18.0, 19.0])
def test_one_key_above_many(dev, high):
    """One key outweighs each of 131071 others by e^high, which together have up to 0.4 % of the weight: every value is 1,
    so out is 1, off by P's rounding of that share, one of the result, and the float32 sums: P v has one addition every
    16 keys, P one every 64, each off by 2^-23 or 2^-24 of the sum (the matrix unit's need not round to the nearest)."""
    n = 1 << 17
    q, k = (torch.zeros((1, n, 1, 64), dtype=torch.float16, device=dev) for _ in range(2))
    q[..., 0] = 1.0
    k[:, 0, :, 0] = high
    v = torch.ones_like(k)
    out, lse = context.window_attention_forward(q, k, v, None, None, scale=1.0)
    top = k[0, 0, 0, 0].double().item()
    share = (n - 1) / (n - 1 + math.exp(top))
    print(f"share {share:.2e} off by {(out.double() - 1).abs().max().item():.2e}", flush=True)
    assert ((out.double() - 1).abs() <= U * (1 + share) + 2.0 ** -23 * n / 16 + 2.0 ** -24 * n / 64).all()
    # (32 more additions in a tile, the logarithm, products)
    assert ((lse.double() - (top + math.log1p((n - 1) * math.exp(-top)))).abs() <= 2.0 ** -24 * (n / 64 + 64 + 4 * top)).all()


@pytest.mark.parametrize("vs", [1e-2, 1e-4, 0.0])
@pytest.mark.parametrize("size", [1e-3, 1e-5, 1e-7])
def test_small_values_and_small_gradients(dev, size, vs):
    """Gradients whose bound is below 2^-16 with values far below 1, to the smallest that float16 holds, and zeros."""
    for n, how in ((2, dict(left=0, right=0)), (500, dict(left=None, right=0)), (300, dict(left=20, right=20, sinks=3))):
        q, k, v, do = _inputs(dev, n, 2, n, 2, 1, 64, size, 3.0, vs)
        got = _check(q, k, v, do, **how)
        assert all(t.isfinite().all() for t in got)
