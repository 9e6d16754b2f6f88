"""AdamW over many tensors on the GPU: to the bit the same as the steps written out in float32 with every operation
rounded by itself, and within float32's rounding of the formula in float64."""
from __future__ import annotations

import math

import pytest
import torch

from rsna_knee_efficiency_amd import densenet, optim

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
LR, B1, B2, EPS, WD, BLOCK = 3e-3, 0.9, 0.99, 1e-8, 0.02, 256


def _blocks(x):
    n = x.numel()
    return torch.cat([x.reshape(-1).float(), x.new_zeros(-n % BLOCK, dtype=F32)])


class Plain:
    """One tensor's step, operation by operation."""

    def __init__(self, p, bits):
        self.p, self.bits, self.t = p.clone(), bits, 0
        n = -(-p.numel() // BLOCK) * BLOCK
        self.m, self.v = torch.zeros(n, device=p.device), torch.zeros(n, device=p.device)

    def step(self, g, scale=None):
        self.t += 1
        g = _blocks(g)
        g = g * scale if scale is not None else g
        m = self.m * B1 + g * (1 - B1)
        v = self.v * B2 + g * g * (1 - B2)
        r = v.sqrt()
        p = _blocks(self.p) * (1 - LR * WD) - m / (r * (1 / math.sqrt(1 - B2 ** self.t)) + EPS) * (LR / (1 - B1 ** self.t))
        self.p = p[:self.p.numel()].view(self.p.shape).to(self.p.dtype)
        if self.bits == 8:
            m, r = m.view(-1, BLOCK), r.view(-1, BLOCK)
            ms, rs = (torch.where(x.abs().amax(1) >= 2.0 ** -100, x.abs().amax(1), 0.0)[:, None] for x in (m, r))
            mi, ri = (torch.where(x > 0, 1 / x, 0.0) for x in (ms, rs))
            c = ((m.abs() * mi).sqrt() * 127).round().clamp(max=127) * m.sign()
            d = ((r * ri).sqrt() * 255).round().clamp(max=255)
            d = torch.where((d == 0) & (r > 0) & (rs > 0), 1.0, d)
            m = (c * c.abs() * (ms * (1 / 127 ** 2))).view(-1)
            v = (d * d * (rs * (1 / 255 ** 2))).view(-1).square()
        self.m, self.v = m, v


SIZES = [(1,), (3, 85), (256,), (257,), (0,), (16, 16), (7, 300), (1024, 1), (5000,), (64, 3, 7, 7)]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("pt,gt", [(F32, F32), (F32, BF16), (F32, F16), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)])
def test_steps_to_the_bit(dev, bits, pt, gt):
    g = torch.Generator(device=dev).manual_seed(3)
    params = [torch.randn(s, generator=g, device=dev).to(pt) for s in SIZES]
    plain = [Plain(p, bits) for p in params]
    opt = optim.AdamW(params, LR, (B1, B2), EPS, WD, bits)
    for t in range(5):
        print(f"adamw {bits} {pt} {gt} step {t}", flush=True)
        grads = [(torch.randn(s, generator=g, device=dev) * 10.0 ** (t - 3)).to(gt) for s in SIZES]
        scale = torch.tensor(0.5 + t, device=dev) if t >= 3 else None
        opt.step(grads, scale)
        for q, x in zip(plain, grads):
            q.step(x, scale)
        assert all(torch.equal(p, q.p) for p, q in zip(params, plain))
        m, v = opt.moments()
        assert torch.equal(m, torch.cat([q.m for q in plain])) and torch.equal(v, torch.cat([q.v for q in plain]))


@pytest.mark.parametrize("bits", [32, 8])
def test_against_float64(dev, bits):
    """Three steps.  float32: each operation is off by 2^-24 of its result, about 16 in a step's chain.  The first
    step of 8-bit moments comes from zeros, so its new parameters are float32's; what the moments stand for is within
    half a step of their codes: a relative 1 / (2 c) + ... of a value at code c, at most s / 127 (c + 1/4) / 127."""
    g = torch.Generator(device=dev).manual_seed(4)
    p = torch.randn(70001, generator=g, device=dev)
    x = [torch.randn(70001, generator=g, device=dev) * 0.1 for _ in range(3)]
    q, m, v = p.double(), torch.zeros(70001, dtype=torch.float64, device=dev), torch.zeros(70001, dtype=torch.float64, device=dev)
    opt = optim.AdamW([p], LR, (B1, B2), EPS, WD, bits)
    for t in range(1, 4 if bits == 32 else 2):
        gd = x[t - 1].double()
        m, v = B1 * m + (1 - B1) * gd, B2 * v + (1 - B2) * gd ** 2
        q = q * (1 - LR * WD) - LR * (m / (1 - B1 ** t)) / ((v / (1 - B2 ** t)).sqrt() + EPS)
        opt.step([x[t - 1]])
        # (sqrt(v) of a gradient near 0 beside eps: the quotient is bounded by sqrt(1 / (1 - B2)) / ... < 20)
        assert ((p.double() - q).abs() <= 2.0 ** -24 * (4 * t * q.abs() + 32 * t * LR * 20)).all()
    gm, gv = (s[:70001].double() for s in opt.moments())
    if bits == 32:
        assert ((gm - m).abs() <= 2.0 ** -24 * 16 * 0.1 * 6).all() and ((gv - v).abs() <= 2.0 ** -24 * 16 * v + 1e-45).all()
        return
    pad = torch.zeros(-70001 % BLOCK, dtype=torch.float64, device=dev)
    for got, want, top in ((gm, m, 127), (gv.sqrt(), v.sqrt(), 255)):
        s = torch.cat([want, pad]).view(-1, BLOCK).abs().amax(1).repeat_interleave(BLOCK)[:70001]
        c = (want.abs() / s).sqrt() * top
        # rounding c to whole codes moves c^2 by at most c + 1/4 (a value raised to code 1: by at most 1)
        assert ((got - want).abs() <= s / top ** 2 * (c + 1.0) * (1 + 2.0 ** -18)).all()


def test_many_tensors_of_a_network(dev):
    """Every parameter of the float DenseNet169 (507 tensors, several launches), some without a gradient."""
    net = densenet.DenseNet().to(dev)
    params = [p.detach() for p in net.parameters()]
    assert len(params) > 300
    g = torch.Generator(device=dev).manual_seed(5)
    grads = [None if i % 50 == 7 else torch.randn(p.shape, generator=g, device=dev) for i, p in enumerate(params)]
    plain = [Plain(p, 32) for p in params]
    opt = optim.AdamW(params, LR, (B1, B2), EPS, WD)
    for _ in range(2):
        opt.step(grads)
        for q, x in zip(plain, grads):
            if x is not None:
                q.step(x)
    assert all(torch.equal(p, q.p) for p, q in zip(params, plain))
    assert torch.equal(opt.moments()[0], torch.cat([q.m for q in plain]))


def test_mixed_types_views_and_grad_attribute(dev):
    """Parameters of two types in one call, at odd addresses, with transposed gradients and gradients in .grad."""
    g = torch.Generator(device=dev).manual_seed(6)
    a = torch.randn(1 + 40 * 30, generator=g, device=dev)[1:].view(40, 30)
    b = torch.randn(1 + 500, generator=g, device=dev).to(BF16)[1:]
    a, b = a.detach().requires_grad_(), b.detach().requires_grad_()
    plain = [Plain(a.detach(), 8), Plain(b.detach(), 8)]
    opt = optim.AdamW([a, b], LR, (B1, B2), EPS, WD, 8)
    ga, gb = torch.randn((30, 40), generator=g, device=dev).t(), torch.randn(500, generator=g, device=dev).to(BF16)
    a.grad, b.grad = ga, gb
    version = a._version
    opt.step()
    plain[0].step(ga.contiguous())
    plain[1].step(gb)
    assert torch.equal(a, plain[0].p) and torch.equal(b, plain[1].p) and a._version > version
    opt.zero_grad()
    assert a.grad is None
    opt.step()                                 # nothing has a gradient: nothing changes
    assert torch.equal(a, plain[0].p) and opt.step_count == 2


def test_state_travels_and_non_finite_gradients_stay_apart(dev):
    g = torch.Generator(device=dev).manual_seed(7)
    p = [torch.randn(600, generator=g, device=dev), torch.randn(10, generator=g, device=dev)]
    x = [torch.randn(600, generator=g, device=dev), torch.randn(10, generator=g, device=dev)]
    for bits in (8, 32):
        a = [t.clone() for t in p]
        one = optim.AdamW(a, LR, (B1, B2), EPS, WD, bits)
        one.step(x)
        b = [t.clone() for t in a]
        two = optim.AdamW(b, LR, (B1, B2), EPS, WD, bits)
        two.load_state_dict(one.state_dict())
        one.step(x)
        two.step(x)
        assert all(torch.equal(s, t) for s, t in zip(a, b)) and all(torch.equal(s, t) for s, t in zip(one.moments(), two.moments()))
        with pytest.raises(ValueError):
            two.load_state_dict({"step": 1})
        bad = [x[0].clone(), x[1]]
        bad[0][300] = float("nan")
        one.step(bad)
        two.step(x)
        fine = torch.ones(600, dtype=torch.bool, device=dev)
        fine[300] = False
        assert torch.equal(a[0][fine], b[0][fine]) and torch.equal(a[1], b[1]) and a[0][300].isnan()
        m, other = one.moments()[0], two.moments()[0]
        spoiled = m.isnan()
        assert torch.equal(m[~spoiled], other[~spoiled])
        assert int(spoiled.sum()) == (1 if bits == 32 else BLOCK) and spoiled[256:512].any()


def test_zero_and_tiny_gradients(dev):
    """All zeros: moments stay zeros and p only decays; values below what a block can be divided by become zeros."""
    p = torch.full((300,), 2.0, device=dev)
    opt = optim.AdamW([p], LR, (B1, B2), EPS, WD, 8)
    opt.step([torch.zeros(300, device=dev)])
    assert torch.equal(p, torch.full((300,), 2.0, device=dev) * (1 - LR * WD))
    assert not any(t.any() for t in opt.moments())
    opt.step([torch.full((300,), 1e-35, device=dev)])
    assert p.isfinite().all() and not any(t.any() for t in opt.moments())


def test_refusals(dev):
    p = torch.zeros((4, 4), device=dev)
    opt = optim.AdamW([p])
    for grads, match in (([torch.zeros((4, 5), device=dev)], "shape"), ([torch.zeros((4, 4))], "device"), ([], "every"),
                         ([torch.zeros((4, 4), device=dev, dtype=torch.float64)], "float64")):
        with pytest.raises(ValueError, match=match):
            opt.step(grads)
    with pytest.raises(ValueError, match="grad_scale"):
        opt.step([p], torch.ones(1))
    with pytest.raises(ValueError, match="contiguous"):
        optim.AdamW([p[:, :2]])
    with pytest.raises(ValueError, match="beside"):
        optim.AdamW([p.half()]).step([p.bfloat16()])
    assert opt.step_count == 0
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="graph"):
            opt.step([torch.zeros_like(p)])
        p.add_(0)
