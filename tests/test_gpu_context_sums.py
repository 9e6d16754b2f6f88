"""Sums of the context layer's operators where a mistake would hide in a looser bound: layer norm's weights' gradients over
several turns of a workgroup in 16 bits, at widths whose last vector overlaps the one before it; attention's lse."""
from __future__ import annotations

import math

import pytest
import torch

from rsna_knee_efficiency_amd import context

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
BF16, F16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("rows,width", [(70001, 7), (40011, 100), (33001, 127), (20003, 300), (9001, 511), (17003, 257),
                                        (9002, 1001), (5003, 2047), (2050, 4097), (1100, 8195)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_layer_norm_columns_over_several_turns(dev, rows, width, dtype):
    """Gradients of one sign: a column left out or counted twice in one turn is a whole share of its sum.  float32
    addition of n terms is off by at most n 2^-24 of their sum; a workgroup adds rows / 1024 of a column, the second
    launch 128, and xh itself is off by 2^-24 (the mean's 64 additions, the centring, rstd) of 1 + |xh| + |mean| / sd
    times 100."""
    g = torch.Generator(device=dev).manual_seed(rows)
    x = (torch.randn((rows, width), generator=g, device=dev) + 0.5).to(dtype)
    dy = torch.rand((rows, width), generator=g, device=dev).to(dtype)
    w = torch.rand(width, generator=g, device=dev) + 0.5
    y, mean, rstd = context.layer_norm_forward(x, w)
    dx, dw, db = context.layer_norm_backward(dy, x, w, mean, rstd)
    x64, dy64 = x.double(), dy.double()
    mu = x64.mean(1, keepdim=True)
    r = ((x64 - mu).square().mean(1, keepdim=True) + 1e-5).rsqrt()
    xh = (x64 - mu) * r
    add = (rows / 256 + 256) * E
    assert ((db.double() - dy64.sum(0)).abs() <= add * dy64.sum(0)).all()
    exh = 100 * E * (1 + xh.abs() + (mu * r).abs()) * (1 + xh.abs())
    assert ((dw.double() - (dy64 * xh).sum(0)).abs() <= (dy64 * (add * xh.abs() + exh)).sum(0)).all()
    # and the rows: y and dx, every column of them
    u = {BF16: 2.0 ** -8, F16: 2.0 ** -11}[dtype]
    step = {BF16: 0.0, F16: 2.0 ** -25}[dtype]
    assert ((y.double() - xh * w.double()).abs() <= u * (xh * w.double()).abs() + 2 * exh * w.double() + step).all()
    z = dy64 * w.double()
    want = r * (z - z.mean(1, keepdim=True) - xh * (z * xh).mean(1, keepdim=True))
    size = r * (z + z.mean(1, keepdim=True) + xh.abs() * (z * xh).abs().mean(1, keepdim=True))
    assert ((dx.double() - want).abs() <= u * want.abs() + 400 * E * (1 + (mu * r).abs()) * (1 + xh.abs()) * size + step).all()


@pytest.mark.parametrize("n,h,hk,d,left,right,sinks,absent,size", [
    (1, 1, 1, 64, None, None, 0, 0.0, 1.5), (77, 2, 1, 128, None, 0, 0, 0.0, 1.5), (700, 4, 2, 64, 100, 20, 3, 0.3, 1.5),
    (2500, 2, 2, 64, None, None, 0, 0.0, 1.5), (2500, 1, 1, 128, 512, 0, 12, 0.2, 1.5), (900, 2, 1, 64, None, 0, 0, 0.0, 30.0),
    (900, 2, 1, 128, 50, 50, 70, 0.5, 30.0)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_statistics_are_float32(dev, n, h, hk, d, left, right, sinks, absent, size, dtype):
    """lse against float64.  A score's d products are added in float32: off by 2 d 2^-24 sum |q k| scale at most, and by
    2^-22 of itself for scale log2(e) and the exponent.  The weights' sum has one addition and, where the maximum
    rises, one factor a tile of 64 keys (2^-23 each), 64 additions within; the logarithm and its products 2^-22."""
    g = torch.Generator(device=dev).manual_seed(n)
    q, k, v = ((torch.randn((2, n, x, d), generator=g, device=dev) * s).to(dtype) for x, s in ((h, size), (hk, 1.0), (hk, 1.0)))
    mask = torch.rand((2, n), generator=g, device=dev) >= absent if absent else None
    _, lse = context.window_attention_forward(q, k, v, left, right, sinks, mask)
    i, j = torch.arange(n, device=dev)[:, None], torch.arange(n, device=dev)[None]
    far = n if left is None else left
    see = (j <= i + (n if right is None else right)) & ((j >= i - far) | (j < sinks))
    see = (see[None] if mask is None else see[None] & mask[:, None])[:, None]
    q, k = q.double().transpose(1, 2), k.double().transpose(1, 2).repeat_interleave(h // hk, 1)
    s = q @ k.transpose(2, 3) / math.sqrt(d)
    off = (2 * d * E * (q.abs() @ k.abs().transpose(2, 3)) / math.sqrt(d) + 2.0 ** -22 * s.abs()).masked_fill(~see, 0.0)
    # an error of every score is one of lse weighted by P: at most the largest, and no more than that of weighty keys
    p = torch.softmax(s.masked_fill(~see, -math.inf), -1).nan_to_num(0.0)
    want = torch.logsumexp(s.masked_fill(~see, -math.inf), -1)
    seen = want.isfinite()
    assert torch.equal(lse.isfinite(), seen) and (lse[~seen] == -math.inf).all()
    bound = 1.01 * (p * off).sum(-1) + (n / 64 + 64) * 2.0 ** -23 + 2.0 ** -22 * want.abs()
    far_off = ((lse.double() - want).abs() / bound)[seen].max().item()
    print(f"lse: {far_off:.2f} of its bound, which is {bound[seen].max().item():.1e} at most", flush=True)
    assert far_off <= 1
