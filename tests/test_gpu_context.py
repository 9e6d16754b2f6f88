"""Layer norm and rotary positions on the GPU against their formulas in float64.

Tolerances: float32 sums of n terms are off by at most n 2^-24 of the sum of the terms' magnitudes, in the order the
kernels add them; a value rounded to bfloat16 (float16) is off by at most 2^-9 (2^-12) of itself, doubled here because
the value before it was rounded may already lie beside a tie."""
from __future__ import annotations

import pytest
import torch

from rsna_knee_efficiency_amd import context

pytestmark = pytest.mark.gpu

EPS32 = 2.0 ** -24
UNIT = {torch.float32: 2.0 ** -23, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -24}
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _norm64(x, w, b, dy, eps):
    x, w, dy = x.double(), w.double(), dy.double()
    mean = x.mean(-1, keepdim=True)
    var = (x - mean).square().mean(-1, keepdim=True)
    r = (var + eps).rsqrt()
    xh = (x - mean) * r
    y = xh * w + (b.double() if b is not None else 0.0)
    g = dy * w
    dx = r * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    return y, dx, (dy * xh).sum(0), dy.sum(0), xh, mean, r, g


def _check_norm(x, w, b, dy, eps=1e-5):
    y, mean, rstd = context.layer_norm_forward(x, w, b, eps)
    dx, dw, db = context.layer_norm_backward(dy, x, w, mean, rstd)
    ry, rdx, rdw, rdb, xh, rmean, rr, g = _norm64(x, w, b, dy, eps)
    n, width = x.shape
    unit = UNIT[x.dtype]
    # a mean of `width` terms in lanes of at most 32 terms, then trees: at most 64 roundings of its terms' magnitude
    emean = 64 * EPS32 * x.double().abs().mean(-1, keepdim=True)
    assert ((mean[:, None].double() - rmean).abs() <= emean).all()
    # xh: the mean's error and the centring's rounding over the row's deviation, twice (in the deviation too)
    exh = 2 * (emean + EPS32 * x.double().abs()) * rr * (1 + xh.abs()) + 96 * EPS32 * xh.abs()
    wm = w.double().abs()
    ey = exh * wm + 4 * EPS32 * ry.abs() + unit * ry.abs() + TINY[x.dtype]
    assert ((y.double() - ry).abs() <= ey).all()
    em = 96 * EPS32 * (g.abs().mean(-1, keepdim=True) + xh.abs() * (g * xh).abs().mean(-1, keepdim=True))
    em = em + (exh * g.abs()).mean(-1, keepdim=True) * xh.abs() + exh * (g * xh).abs().mean(-1, keepdim=True)
    edx = rr * (em + 8 * EPS32 * g.abs()) + rdx.abs() * (exh.amax(-1, keepdim=True) + 96 * EPS32 + unit) + TINY[x.dtype]
    assert ((dx.double() - rdx).abs() <= edx).all()
    add = (n / 4 + 128) * EPS32
    ew = (exh * dy.double().abs()).sum(0) + add * (dy.double() * xh).abs().sum(0) + UNIT[w.dtype] * rdw.abs() + TINY[w.dtype]
    assert ((dw.double() - rdw).abs() <= ew).all()
    eb = add * dy.double().abs().sum(0) + UNIT[w.dtype] * rdb.abs() + TINY[w.dtype]
    assert ((db.double() - rdb).abs() <= eb).all()
    assert y.dtype == dx.dtype == x.dtype and dw.dtype == db.dtype == w.dtype


WIDTHS = [1, 2, 5, 16, 63, 64, 100, 128, 129, 256, 511, 513, 1024, 1025, 1664, 2048, 2049, 4096, 4100, 8191, 8193, 16383,
          16384]


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype,wtype", [(F32, F32), (BF16, F32), (BF16, BF16), (F16, F32), (F16, F16)])
def test_layer_norm(dev, width, dtype, wtype):
    g = torch.Generator(device=dev).manual_seed(width)
    for rows in (1, 3, 17, 70):
        print(f"norm rows={rows} width={width} {dtype} {wtype}", flush=True)
        x = (torch.randn((rows, width), generator=g, device=dev) * 1.5 + 0.3).to(dtype)
        dy = torch.randn((rows, width), generator=g, device=dev).to(dtype)
        w = (torch.randn(width, generator=g, device=dev) * 0.2 + 1).to(wtype)
        b = torch.randn(width, generator=g, device=dev).to(wtype)
        _check_norm(x, w, b, dy)


@pytest.mark.parametrize("rows,width", [(20011, 96), (9001, 256), (5003, 1030), (2001, 2500)])
def test_layer_norm_many_rows(dev, rows, width):
    """More rows than the backward pass has workgroups: each sums several."""
    g = torch.Generator(device=dev).manual_seed(rows)
    x, dy = (torch.randn((rows, width), generator=g, device=dev) for _ in range(2))
    w, b = torch.rand(width, generator=g, device=dev), torch.rand(width, generator=g, device=dev)
    _check_norm(x, w, b, dy)


def test_layer_norm_strides_mean_and_constant_rows(dev):
    """Rows apart, at odd addresses and in two leading dimensions; a mean far larger than the deviation; rows of one
    value (variance 0); no bias; no rows; equal bits from call to call."""
    g = torch.Generator(device=dev).manual_seed(5)
    base = torch.randn((40, 301), generator=g, device=dev)
    x, dy = base[:, 1:258], base.flip(0)[:, 40:297]
    w = torch.rand(257, generator=g, device=dev)
    _check_norm(x, w, None, dy)
    _check_norm(x.to(BF16), w, None, dy.to(BF16))
    _check_norm(base.to(BF16)[:, 3:260], w, None, dy.to(BF16))
    _check_norm(x + 1000.0, w, w, dy)
    const = torch.full((6, 257), 3.25, device=dev)
    y, mean, rstd = context.layer_norm_forward(const, w, w)
    assert torch.equal(y, w.expand_as(y)) and torch.equal(mean, const[:, 0])
    nd = base[:, :256].reshape(5, 8, 256)
    a = context.layer_norm(nd, w[:256], None)
    assert a.shape == nd.shape and torch.equal(a.view(40, 256), context.layer_norm(base[:, :256], w[:256], None))
    swapped = nd.transpose(0, 1)
    assert torch.equal(context.layer_norm(swapped, w[:256]), a.transpose(0, 1))
    empty = torch.zeros((0, 257), device=dev)
    y, m, r = context.layer_norm_forward(empty, w)
    dx, dw, db = context.layer_norm_backward(empty, empty, w, m, r)
    assert y.shape == dx.shape == (0, 257) and not dw.any() and not db.any()
    first = context.layer_norm_backward(dy, x, w, *context.layer_norm_forward(x, w)[1:])
    again = context.layer_norm_backward(dy, x, w, *context.layer_norm_forward(x, w)[1:])
    assert all(torch.equal(p, q) for p, q in zip(first, again))


def test_layer_norm_gradient_by_differences(dev):
    """Central differences of the formula in float64 along random directions: step 1e-4, whose own error is about 1e-8
    of the derivative; the float32 gradients are within 1e-4 of the sum of their terms' magnitudes."""
    g = torch.Generator(device=dev).manual_seed(6)
    x, dy = (torch.randn((9, 83), generator=g, device=dev) for _ in range(2))
    w, b = (torch.randn(83, generator=g, device=dev) for _ in range(2))
    xs, ws, bs = (t.clone().requires_grad_() for t in (x, w, b))
    (context.layer_norm(xs, ws, bs) * dy).sum().backward()

    def loss(x, w, b):
        return (_norm64(x, w, b, dy, 1e-5)[0] * dy.double()).sum()
    for leaf, at in ((xs, 0), (ws, 1), (bs, 2)):
        d = torch.randn(leaf.shape, generator=g, device=dev, dtype=torch.float64)
        args = [x.double(), w.double(), b.double()]
        up, down = list(args), list(args)
        up[at], down[at] = args[at] + 1e-4 * d, args[at] - 1e-4 * d
        want = (loss(*up) - loss(*down)) / 2e-4
        got = (leaf.grad.double() * d).sum()
        assert abs(got - want) <= 1e-4 * (leaf.grad.double() * d).abs().sum()


def test_layer_norm_keeps_non_finite_rows_apart(dev):
    x = torch.randn((40, 300), device=dev)
    want = context.layer_norm(x, torch.ones(300, device=dev))
    x[7, 3], x[21, 299] = float("nan"), float("inf")
    got = context.layer_norm(x, torch.ones(300, device=dev))
    bad = torch.zeros(40, dtype=torch.bool, device=dev)
    bad[7] = bad[21] = True
    assert torch.equal(got[~bad], want[~bad]) and got[bad].isnan().all()


# --- rotary positions ---------------------------------------------------------------------------------
def _rotary64(x, pos, sections, base, adjacent, inverse):
    x = x.double().clone()
    n = sum(sections)
    turn, axis = [], []
    for a, s in enumerate(sections):
        for t in range(s):
            turn.append(base ** (-t / s))
            axis.append(a)
    pos = pos.double() if pos.dim() == 3 else pos.double()[None]
    angle = (pos[..., axis] * torch.tensor(turn, dtype=torch.float64, device=x.device))[:, :, None]
    c, s = angle.cos(), angle.sin() * (-1 if inverse else 1)
    i = slice(0, 2 * n, 2) if adjacent else slice(0, n)
    j = slice(1, 2 * n, 2) if adjacent else slice(n, 2 * n)
    u, v = x[..., i].clone(), x[..., j].clone()
    x[..., i], x[..., j] = u * c - v * s, u * s + v * c
    return x


def _check_rotary(x, pos, sections, base=10000.0, adjacent=False, inverse=False, far=0.0):
    got = context.rotary(x, pos, sections, base, adjacent=adjacent, inverse=inverse)
    want = _rotary64(x, pos, sections, base, adjacent, inverse)
    # the angle's turns are rounded to float32 (2^-25 of a turn), sine and cosine to 2 units; two products, one sum;
    # `far`: what float64 itself loses of a large angle in the oracle's own sine
    size = x.double().abs().amax(-1, keepdim=True) * 2
    tol = size * (2 ** -25 * 6.3 + 6 * EPS32 + far) + UNIT[x.dtype] * want.abs() + TINY[x.dtype]
    assert got.dtype == x.dtype and ((got.double() - want).abs() <= tol).all()
    n = 2 * sum(sections)
    assert torch.equal(got[..., n:], x[..., n:])


@pytest.mark.parametrize("dim,sections", [(2, (1,)), (6, (1, 2)), (16, (8,)), (20, (3, 2, 4)), (64, (8, 12, 12)),
                                          (64, (5, 0, 7)), (67, (10, 10, 10)), (128, (16, 24, 24)), (130, (65,)),
                                          (512, (100, 100, 56))])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_rotary(dev, dim, sections, dtype):
    g = torch.Generator(device=dev).manual_seed(dim)
    for b, s, h in ((1, 1, 1), (2, 7, 3), (3, 129, 5)):
        print(f"rotary {b} {s} {h} {dim} {sections} {dtype}", flush=True)
        x = torch.randn((b, s, h, dim), generator=g, device=dev).to(dtype)
        pos = torch.randint(-50, 300, (b, s, len(sections)), generator=g, device=dev)
        for adjacent in (False, True):
            for inverse in (False, True):
                _check_rotary(x, pos.int(), sections, 10000.0, adjacent, inverse)
        _check_rotary(x, pos[0], sections, 100.0)
        _check_rotary(x, pos.float() + 0.25, sections)


def test_rotary_positions_far_out(dev):
    """Positions of millions, and of the last an int32 holds, turn as exactly as small ones (the oracle's angle,
    rounded to 53 bits, is off by 2^-53 of itself)."""
    g = torch.Generator(device=dev).manual_seed(9)
    x = torch.randn((1, 50, 2, 64), generator=g, device=dev)
    pos = torch.randint(0, 1 << 22, (50, 2), generator=g, device=dev)
    _check_rotary(x, pos, (16, 16), far=2.0 ** -53 * (1 << 22) * 4)
    pos = torch.full((50, 2), 2 ** 31 - 1, device=dev, dtype=torch.int32) - torch.arange(50, device=dev, dtype=torch.int32)[:, None]
    _check_rotary(x, pos, (16, 16), far=2.0 ** -53 * 2.0 ** 31 * 4)


def test_rotary_strides_in_place_and_gradient(dev):
    g = torch.Generator(device=dev).manual_seed(10)
    packed = torch.randn((2, 60, 3, 4, 64), generator=g, device=dev).to(BF16)
    pos = torch.randint(0, 40, (2, 60, 3), generator=g, device=dev, dtype=torch.int32)
    qk = packed[:, :, :2].flatten(2, 3)                     # queries and keys beside each other: a view
    assert qk.data_ptr() == packed.data_ptr()
    _check_rotary(qk, pos, (8, 12, 12))
    _check_rotary(packed[:, :, 1].transpose(1, 2).contiguous().transpose(1, 2), pos, (8, 12, 12))
    _check_rotary(packed.reshape(-1)[1:1 + 2 * 30 * 2 * 64].view(2, 30, 2, 64), pos[:, :30], (8, 12, 12))
    _check_rotary(qk, pos.flip(-1), (8, 12, 12))
    spread = torch.randn((2, 60, 4, 128), generator=g, device=dev)[..., ::2]
    _check_rotary(spread, pos, (8, 12, 12))
    want = context.rotary(qk, pos, (8, 12, 12))
    values = packed[:, :, 2].clone()
    version = packed._version
    assert context.rotary(qk, pos, (8, 12, 12), out=qk).data_ptr() == packed.data_ptr()
    assert torch.equal(qk, want) and torch.equal(packed[:, :, 2], values) and packed._version > version
    x = torch.randn((2, 60, 4, 64), generator=g, device=dev, requires_grad=True)
    dy = torch.randn((2, 60, 4, 64), generator=g, device=dev)
    y = context.rotary(x, pos, (8, 12, 10), adjacent=True)
    y.backward(dy)
    assert torch.equal(x.grad, context.rotary(dy, pos, (8, 12, 10), adjacent=True, inverse=True))
    back = context.rotary(y.detach(), pos, (8, 12, 10), adjacent=True, inverse=True)
    assert ((back - x).abs() <= 32 * EPS32 * x.abs().amax()).all()
    d = torch.randn(x.shape, generator=g, device=dev, dtype=torch.float64)
    up, down = (_rotary64(x.detach().double() + s * d, pos, (8, 12, 10), 10000.0, True, False) for s in (1e-4, -1e-4))
    want = ((up - down) * dy.double()).sum() / 2e-4
    assert abs((x.grad.double() * d).sum() - want) <= 1e-5 * (x.grad.double() * d).abs().sum()
    assert context.rotary(x.detach()[:, :0], pos[:, :0], (8, 12, 12)).shape == (2, 0, 4, 64)
    with pytest.raises(ValueError, match="out"):
        context.rotary(x, pos, (8, 12, 12), out=torch.empty_like(x))
    square = torch.randn((4, 4, 1, 8), generator=g, device=dev)
    with pytest.raises(ValueError, match="memory of its own"):
        context.rotary(square, pos[0, :4, :1], (4,), out=square.transpose(0, 1))
