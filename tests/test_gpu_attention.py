"""Attention within a window and first tokens on the GPU, with its gradients and the form for one new token, against
the formulas in float64 on the values the 16-bit tensors hold.

Tolerances follow what the kernels round: P and dS to 16 bits before the second product (u = 2^-9 or 2^-12 of each),
results to 16 bits, and scores in float32 (an error es = 2 D 2^-24 sum |q k| scale of s is the same relative error
of P).  Every bound is a sum of magnitudes formed in the oracle with the same weights as the result; twice u is
allowed where a value is rounded after an already rounded one."""
from __future__ import annotations

import math

import pytest
import torch

from rsna_knee_efficiency_amd import context

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
U = {BF16: 2.0 ** -8, F16: 2.0 ** -11}
# what a P too small to hold may be off by: float16's smallest step; float32's smallest normal number (its exp is 0 below)
TINY = {BF16: 2.0 ** -126, F16: 2.0 ** -24}


def _seen(n, left, right, sinks, mask, dev):
    i, j = torch.arange(n, device=dev)[:, None], torch.arange(n, device=dev)[None]
    left, right = n if left is None else left, n if right is None else right
    see = (j <= i + right) & ((j >= i - left) | (j < sinks))
    return see[None] if mask is None else see[None] & mask.bool()[:, None]


def _oracle(q, k, v, dout, left, right, sinks, mask, scale):
    """(out, lse, dq, dk, dv) in float64, and the bounds of all but lse"""
    u, tiny = U[q.dtype], TINY[q.dtype]
    b, n, h, d = q.shape
    per = h // k.shape[2]
    see = _seen(n, left, right, sinks, mask, q.device)[:, None]                            # (b, 1, n, n)
    q, k, v, do = (t.double().transpose(1, 2) for t in (q, k, v, dout))
    if mask is not None:                                    # whatever lies there is not used
        k, v = (t.masked_fill(~mask.bool()[:, None, :, None], 0.0) for t in (k, v))
    k, v = (t.repeat_interleave(per, 1) for t in (k, v))
    s = q @ k.transpose(2, 3) * scale
    es = 2 * d * 2.0 ** -24 * (q.abs() @ k.abs().transpose(2, 3)).amax() * scale + 2.0 ** -19
    s = s.masked_fill(~see, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.where(see, torch.exp(s - torch.where(lse.isfinite(), lse, 0.0)[..., None]), 0.0)
    o = p @ v
    e = (u + 2 * es) * (p @ v.abs()) + u * o.abs() + tiny * (1 + see.double() @ v.abs())
    # gradients; what the kernels keep of o is rounded, so rowsum(do o) is off by u sum |do o|
    dp, row = do @ v.transpose(2, 3), (do * o).sum(-1, keepdim=True)
    ds = p * (dp - row)
    erow = (u * (do * o).abs() + 2.0 ** -20 * (do * o).abs() + tiny * do.abs()).sum(-1, keepdim=True) + (do.abs() * e).sum(-1, keepdim=True)
    edp = 2 * d * 2.0 ** -24 * (do.abs() @ v.abs().transpose(2, 3))
    eds = (u + 4 * es) * ds.abs() + p * (erow + edp) + (tiny + 2.0 ** -126 * (dp - row).abs()) * see
    dq, dk, dv = ds @ k * scale, ds.transpose(2, 3) @ q * scale, p.transpose(2, 3) @ do
    edq = eds @ k.abs() * scale + u * dq.abs() + tiny
    edk = eds.transpose(2, 3) @ q.abs() * scale
    edv = ((u + 4 * es) * p + tiny * see).transpose(2, 3) @ do.abs()

    def shared(t):                                          # the sum over the query heads of a key head
        return t.reshape(b, -1, per, n, d).sum(2)
    dk, dv = shared(dk), shared(dv)
    edk, edv = shared(edk) + u * dk.abs() + tiny, shared(edv) + u * dv.abs() + tiny
    back = [t.transpose(1, 2) for t in (o, dq, dk, dv, e, edq, edk, edv)]
    return lse, back[:4], back[4:]


def _check(q, k, v, dout, left=None, right=0, sinks=0, mask=None, scale=None):
    how = dict(left=left, right=right, sinks=sinks, key_mask=mask, scale=scale)
    out, lse = context.window_attention_forward(q, k, v, **how)
    got = (out, *context.window_attention_backward(dout, q, k, v, out, lse, **how))
    want_lse, want, tol = _oracle(q, k, v, dout, left, right, sinks, mask, scale or 1 / math.sqrt(q.shape[-1]))
    for name, x, y, e in zip(("out", "dq", "dk", "dv"), got, want, tol):
        off = (x.double() - y).abs()
        assert x.dtype == q.dtype and (off <= e).all(), (name, off.max().item(), (off / e.clamp(min=1e-30)).max().item())
    fine = want_lse.isfinite()
    assert torch.equal(lse.isfinite(), fine) and (lse[~fine] == -math.inf).all()
    assert ((lse.double() - want_lse)[fine].abs() <= 1e-3 * (1 + want_lse[fine].abs())).all()
    assert torch.equal(context.window_attention(q, k, v, **how), out)
    return out


def _inputs(dev, seed, b, n, h, hk, d, dtype, qs=1.5):
    g = torch.Generator(device=dev).manual_seed(seed)
    shapes = ((b, n, h, d), (b, n, hk, d), (b, n, hk, d), (b, n, h, d))
    return [(torch.randn(s, generator=g, device=dev) * (qs if i == 0 else 1.0)).to(dtype) for i, s in enumerate(shapes)]


WINDOWS = [(None, 0, 0), (None, None, 0), (0, 0, 0), (0, 0, 3), (1, 0, 1), (40, 0, 4), (63, 64, 0), (64, 63, 64),
           (100, 7, 70), (5, 130, 1000), (0, 20, 0)]


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 65, 127, 128, 129, 200, 333])
@pytest.mark.parametrize("dtype,d", [(BF16, 64), (F16, 128)])
def test_lengths_and_windows(dev, n, dtype, d):
    q, k, v, do = _inputs(dev, n, 2, n, 2, 2, d, dtype)
    for left, right, sinks in WINDOWS:
        print(f"attention n={n} {dtype} left={left} right={right} sinks={sinks}", flush=True)
        _check(q, k, v, do, left, right, sinks)


@pytest.mark.parametrize("h,hk", [(1, 1), (4, 1), (6, 2), (8, 8), (5, 1), (16, 2)])
@pytest.mark.parametrize("dtype,d", [(F16, 64), (BF16, 128)])
def test_shared_heads(dev, h, hk, dtype, d):
    q, k, v, do = _inputs(dev, 100 + h, 2, 150, h, hk, d, dtype)
    _check(q, k, v, do, 50, 0, 2)
    _check(q, k, v, do, 50, 50, 2, scale=0.3)


@pytest.mark.parametrize("dtype,d", [(BF16, 64), (BF16, 128), (F16, 64)])
def test_masks(dev, dtype, d):
    """Random keys off, whole tiles off, every key off (rows that see nothing: zeros, no gradient), a row's only
    visible keys off; not-a-number and infinity in masked keys and values change nothing."""
    n = 300
    q, k, v, do = _inputs(dev, 7, 3, n, 4, 2, d, dtype)
    g = torch.Generator(device=dev).manual_seed(8)
    mask = torch.rand((3, n), generator=g, device=dev) < 0.6
    mask[1, 64:200] = False
    mask[2] = False
    for left, right, sinks in ((None, 0, 0), (30, 30, 0), (20, 0, 5)):
        clean = _check(q, k, v, do, left, right, sinks, mask)
        assert not clean[2].any()
        bad = [t.clone() for t in (k, v)]
        for t, x in zip(bad, (float("nan"), float("inf"))):
            t[~mask] = x
        how = dict(left=left, right=right, sinks=sinks, key_mask=mask.to(torch.uint8) * 7)
        out, lse = context.window_attention_forward(q, *bad, **how)
        assert torch.equal(out, clean)
        grads = context.window_attention_backward(do, q, *bad, out, lse, **how)
        want = context.window_attention_backward(do, q, k, v, out, lse, **how)
        assert all(torch.equal(a, b) for a, b in zip(grads, want))
        assert not grads[1][~mask].any() and not grads[2][~mask].any() and not grads[0][2].any()


def test_large_scores_and_one_sided_rows(dev):
    """Scores of hundreds (a softmax with one key), and running maxima that rise tile after tile."""
    q, k, v, do = _inputs(dev, 11, 1, 400, 2, 2, 64, BF16, qs=30.0)
    _check(q, k, v, do, None, 0, 0)
    k = k * torch.linspace(0.1, 3, 400, device=dev)[None, :, None, None].to(BF16)
    q = q.abs() * 0.05
    _check(q, k.abs(), v, do, None, None, 0)
    _check(q, -k.abs(), v, do, None, None, 0)


def test_strides(dev):
    """Heads before tokens in memory, queries, keys and values of one packed tensor, odd addresses, keys and gradients
    broadcast over heads or the batch (stride 0), channels apart (copied)."""
    n, d = 130, 64
    q, k, v, do = _inputs(dev, 12, 2, n, 4, 4, d, BF16)
    want = _check(q, k, v, do, 40, 10, 3)
    how = dict(left=40, right=10, sinks=3)

    def both(q, k, v, do):
        out, lse = context.window_attention_forward(q, k, v, **how)
        return (out, *context.window_attention_backward(do, q, k, v, out, lse, **how))
    plain = both(q, k, v, do)
    assert torch.equal(plain[0], want)
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v, do)]
    packed = torch.stack((q, k, v), 2)
    odd = []
    for t in (q, k, v, do):
        buf = torch.empty(t.numel() + 1, dtype=t.dtype, device=dev)[1:].view(t.shape)
        odd.append(buf.copy_(t))
    apart = [torch.stack((t, t), -1)[..., 0] for t in (q, k, v, do)]
    for case in (heads_first, [packed[:, :, 0], packed[:, :, 1], packed[:, :, 2], do], odd, apart):
        assert all(torch.equal(a, b) for a, b in zip(plain, both(*case)))
    one = k[:, :, :1].expand(-1, -1, 4, -1)
    ones = torch.ones((), dtype=BF16, device=dev).expand(q.shape)
    assert all(torch.equal(a, b) for a, b in zip(both(q, one, v, ones), both(q, one.contiguous(), v, ones.contiguous())))
    mask = (torch.arange(2 * n, device=dev) % 5 != 0)[::2].expand(2, n)
    _check(q, k, v, do, 40, 10, 3, mask)


@pytest.mark.parametrize("n,h,hk,d,left,right,sinks", [(2500, 2, 1, 64, 200, 0, 4), (1900, 1, 1, 128, 64, 64, 130),
                                                       (3000, 2, 2, 64, None, None, 1)])
def test_long(dev, n, h, hk, d, left, right, sinks):
    """First tokens whose gradient is split over many runs of queries; few heads, whose tiles are split too."""
    q, k, v, do = _inputs(dev, n, 1, n, h, hk, d, BF16)
    _check(q, k, v, do, left, right, sinks)


def test_empty_and_repeated(dev):
    q, k, v, do = _inputs(dev, 13, 1, 700, 4, 1, 64, F16)
    z = [t[:, :0] for t in (q, k, v, do)]
    out, lse = context.window_attention_forward(*z[:3])
    assert out.shape == (1, 0, 4, 64) and lse.shape == (1, 4, 0)
    assert [g.shape for g in context.window_attention_backward(z[3], *z[:3], out, lse)] == [t.shape for t in z[:3]]
    out, lse = context.window_attention_forward(q, k, v, 100, 0, 4)
    a = context.window_attention_backward(do, q, k, v, out, lse, 100, 0, 4)
    b = context.window_attention_backward(do, q, k, v, out, lse, 100, 0, 4)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_gradient_by_differences(dev):
    """sum(out dout) in float64 along each gradient's own direction, central differences with a step of 2^-5 of the
    inputs' size: its error is that of out's rounding, 2^-11 sqrt(terms) |out dout| / (2 step) against a derivative of
    the gradient's length, plus the third derivative's step^2: below 3 % together."""
    q, k, v, do = _inputs(dev, 14, 1, 100, 2, 1, 64, F16, qs=1.0)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    context.window_attention(*leaves, 30, 5, 2).backward(do)
    for i, leaf in enumerate(leaves):
        d = leaf.grad.double() / leaf.grad.double().norm() * math.sqrt(leaf.numel()) * 2.0 ** -5
        up, down = [q, k, v], [q, k, v]
        up[i], down[i] = (leaf.detach().double() + d).half(), (leaf.detach().double() - d).half()
        moved = up[i].double() - down[i].double()
        a, b = (context.window_attention(*x, 30, 5, 2).double() for x in (up, down))
        want, got = ((a - b) * do.double()).sum(), (leaf.grad.double() * moved).sum()
        assert abs(got - want) <= 0.03 * abs(got), (i, got.item(), want.item())


# --- one new token ----------------------------------------------------------------------------------------
def _token64(q, k, v, lengths, left, sinks, scale):
    out, tol = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    per = q.shape[1] // k.shape[2]
    for b, n in enumerate(lengths.tolist()):
        n = max(0, min(n, k.shape[1]))
        if n == 0:
            continue
        j = torch.arange(n, device=q.device)
        j = j[(j >= n - 1 - (n if left is None else left)) | (j < sinks)]
        kk, vv = (t[b, j].double().repeat_interleave(per, 1) for t in (k, v))
        s = torch.einsum("hd,jhd->hj", q[b].double(), kk) * scale
        es = 2 * q.shape[2] * 2.0 ** -24 * torch.einsum("hd,jhd->hj", q[b].double().abs(), kk.abs()).amax() * scale + 2.0 ** -18
        p = torch.softmax(s, -1)
        out[b] = torch.einsum("hj,jhd->hd", p, vv)
        tol[b] = 4 * es * torch.einsum("hj,jhd->hd", p, vv.abs()) + U[q.dtype] * out[b].abs() + TINY[q.dtype]
    return out, tol


@pytest.mark.parametrize("h,hk", [(1, 1), (2, 1), (3, 1), (4, 2), (8, 1), (10, 1), (32, 4), (17, 1)])
@pytest.mark.parametrize("dtype,d", [(BF16, 64), (F16, 128)])
def test_token(dev, h, hk, dtype, d):
    g = torch.Generator(device=dev).manual_seed(h)
    lengths = torch.tensor([0, 1, 2, 33, 64, 777, 900, 5000, -3], device=dev, dtype=torch.int32)
    cap = 900
    q = (torch.randn((9, h, d), generator=g, device=dev) * 1.5).to(dtype)
    k, v = (torch.randn((9, cap, hk, d), generator=g, device=dev).to(dtype) for _ in range(2))
    for b, n in enumerate(lengths.clamp(0, cap).tolist()):   # what lies past a row's length is not read
        k[b, n:], v[b, n:] = float("nan"), float("inf")
    for left, sinks in ((None, 0), (0, 0), (0, 2), (100, 4), (500, 64), (300, 2000)):
        print(f"token {h} {hk} {d} left={left} sinks={sinks}", flush=True)
        got = context.window_attention_token(q, k, v, lengths, left, sinks)
        want, tol = _token64(q, k, v, lengths, left, sinks, 1 / math.sqrt(d))
        assert ((got.double() - want).abs() <= tol).all(), ((got.double() - want).abs() / tol.clamp(min=1e-30)).max()
        assert not got[0].any() and not got[8].any()


def test_token_is_the_last_row_of_the_whole(dev):
    """The cache's layout with heads first, one row and many; against the whole attention's last row."""
    q, k, v, _ = _inputs(dev, 15, 1, 1500, 8, 2, 64, BF16)
    whole = context.window_attention(q, k, v, 400, 0, 6)
    kc, vc = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))
    for n in (1, 5, 6, 400, 401, 407, 1000, 1500):
        got = context.window_attention_token(q[:, n - 1], kc, vc, torch.tensor([n], device=dev, dtype=torch.int32), 400, 6)
        # both are within u (twice, for P in the whole) of the exact row, whose values are below 4
        assert ((got.double() - whole[:, n - 1].double()).abs() <= 3 * U[BF16] * 4).all()
    many = context.window_attention_token(q[0, :300].contiguous(), kc.expand(300, -1, -1, -1), vc.expand(300, -1, -1, -1),
                                          torch.arange(1, 301, device=dev, dtype=torch.int32), 400, 6)
    assert ((many.double() - whole[0, :300].double()).abs() <= 3 * U[BF16] * 4).all()
    assert context.window_attention_token(q[:0, 0], k[:0], v[:0], torch.zeros(0, device=dev, dtype=torch.int32)).shape == (0, 8, 64)


def test_offsets_past_32_bits(dev):
    """Rows so far apart that element offsets pass 2^31 (one buffer of 5 GB holds keys, values and queries)."""
    n, step = 620, 4 << 20
    buf = torch.empty(n * step, dtype=BF16, device=dev)
    far = buf.as_strided((1, n, 3, 64), (0, step, 64, 1))
    q, k, v, do = _inputs(dev, 16, 1, n, 1, 1, 64, BF16)
    for i, t in enumerate((q, k, v)):
        far[:, :, i:i + 1].copy_(t)
    fq, fk, fv = (far[:, :, i:i + 1] for i in range(3))
    assert (n - 1) * step > 2 ** 31
    out, lse = context.window_attention_forward(q, k, v, 200, 0, 4)
    got, got_lse = context.window_attention_forward(fq, fk, fv, 200, 0, 4)
    assert torch.equal(out, got) and torch.equal(lse, got_lse)
    a = context.window_attention_backward(do, q, k, v, out, lse, 200, 0, 4)
    b = context.window_attention_backward(do, fq, fk, fv, out, lse, 200, 0, 4)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    length = torch.tensor([n], device=dev, dtype=torch.int32)
    assert torch.equal(context.window_attention_token(q[:, -1], k, v, length, 200, 4),
                       context.window_attention_token(q[:, -1], fk, fv, length, 200, 4))


def test_streams_and_graphs(dev):
    """On another stream, and recorded: every replay gives the eager result on the inputs of the moment."""
    q, k, v, do = _inputs(dev, 17, 1, 500, 4, 2, 64, BF16)
    w = torch.rand(64, device=dev)

    def step():
        x = context.layer_norm(q, w)
        out, lse = context.window_attention_forward(x, k, v, 100, 20, 3)
        grads = context.window_attention_backward(do, x, k, v, out, lse, 100, 20, 3)
        token = context.window_attention_token(x[:, -1], k, v, lengths, 100, 3)
        y, m, r = context.layer_norm_forward(grads[0], w)
        return (out, *grads, token, y, *context.layer_norm_backward(do, grads[0], w, m, r))
    lengths = torch.tensor([480], device=dev, dtype=torch.int32)
    want = step()
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    for i in range(3):
        q.copy_(torch.randn(q.shape, device=dev))
        do.copy_(torch.randn(do.shape, device=dev))
        graph.replay()
        torch.cuda.synchronize(dev)
        assert all(torch.equal(a, b) for a, b in zip(step(), kept)), i
