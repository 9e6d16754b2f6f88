"""The context layer: the operators together, against the same layer written out in float32, one token at a time against
whole studies, and in training."""
from __future__ import annotations

import math

import pytest
import torch

from rsna_knee_efficiency_amd.context_layer import ContextLayer, TokenCache, study_positions, train

pytestmark = pytest.mark.gpu


def _rounded(x):
    return x.bfloat16().float()


def _plain(layer: ContextLayer, w: dict, x, positions, mask, open_units):
    """The layer in float32, its weights rounded to bfloat16 as the layer rounds them, with the hidden units that were
    open in the layer (one whose sign a rounding turns is no rounding error of the gradient, but another function)"""
    def norm(x, a, b):
        c = x - x.mean(-1, keepdim=True)
        return c * (c.square().mean(-1, keepdim=True) + 1e-5).rsqrt() * a + b

    def linear(x, n):
        return x @ w[n + "_w"].bfloat16().float().T + w[n + "_b"]
    b, n, _ = x.shape
    h, hk = layer.heads, layer.key_heads
    qkv = linear(norm(x, w["ln1_w"], w["ln1_b"]), "qkv").view(b, n, h + 2 * hk, 64)
    freq = torch.cat([10000.0 ** (-torch.arange(s, device=x.device, dtype=torch.float64) / s) for s in layer.sections])
    axis = [a for a, s in enumerate(layer.sections) for _ in range(s)]
    angle = positions.double()[..., axis] * freq
    c, s = angle.cos().float()[..., None, :], angle.sin().float()[..., None, :]
    qk = qkv[:, :, :h + hk]
    u, v = qk[..., :32], qk[..., 32:]
    qk = torch.cat([u * c - v * s, u * s + v * c], -1)
    q, k, v = qk[:, :, :h], qk[:, :, h:].repeat_interleave(h // hk, 2), qkv[:, :, h + hk:].repeat_interleave(h // hk, 2)
    i, j = torch.arange(n, device=x.device)[:, None], torch.arange(n, device=x.device)[None]
    left, right = (n if side is None else side for side in (layer.left, layer.right))
    see = ((j <= i + right) & ((j >= i - left) | (j < layer.sinks)))[None, None] & mask[:, None, None]
    p = torch.softmax((q.transpose(1, 2) @ k.permute(0, 2, 3, 1) / 8).masked_fill(~see, -math.inf), -1)
    o = (p @ v.transpose(1, 2)).transpose(1, 2).reshape(b, n, -1)
    x = x + linear(o, "out")
    return x + linear(linear(norm(x, w["ln2_w"], w["ln2_b"]), "ff1") * open_units, "ff2")


def test_layer_and_its_gradients(dev, monkeypatch):
    """About eight results of the chain are rounded to bfloat16 (2^-9 of each), most of them twice in a gradient: the
    outputs within 2 % and the gradients within 4 % of the float32 layer's, by their norms."""
    layer = ContextLayer(heads=4, key_heads=2, left=60, right=40, sinks=5, device=dev)
    positions = study_positions(5, 6, 7, 5, dev)
    n = positions.shape[0]
    g = torch.Generator(device=dev).manual_seed(1)
    x = _rounded(torch.randn((2, n, 256), generator=g, device=dev)).requires_grad_()
    dy = _rounded(torch.randn((2, n, 256), generator=g, device=dev))
    mask = torch.rand((2, n), generator=g, device=dev) < 0.8
    mask[:, :5] = True
    relu, seen = torch.relu, []
    monkeypatch.setattr(torch, "relu", lambda t: (seen.append(t.detach() > 0), relu(t))[1])
    y = layer(x, positions, mask)
    y.backward(dy.bfloat16())
    got = [x.grad, *(p.grad for p in layer.params)]
    x2 = x.detach().clone().requires_grad_()
    w = {k: t.detach().clone().requires_grad_() for k, t in layer.w.items()}
    z = _plain(layer, w, x2, positions, mask, seen[0])
    z.backward(dy)
    assert (y.float() - z).norm() <= 0.02 * z.norm()
    for name, a, b in zip(["x", *w], got, [x2.grad, *(t.grad for t in w.values())]):
        assert (a.float() - b).norm() <= 0.04 * b.norm(), name


def test_one_token_at_a_time(dev):
    """Tokens in order of arrival give the whole study's rows: both are within 2 % of float32's (above), so within 4 %
    of each other."""
    layer = ContextLayer(heads=4, key_heads=1, left=50, right=0, sinks=4, device=dev)
    positions = study_positions(4, 5, 6, 4, dev)
    n = positions.shape[0]
    x = torch.randn((3, n, 256), device=dev).bfloat16()
    with torch.no_grad():
        whole = layer(x, positions)
    cache = TokenCache(layer, 3, n)
    rows = torch.stack([layer.token(x[:, i], positions[i].expand(3, 3), cache) for i in range(n)], 1)
    assert (rows.float() - whole.float()).norm() <= 0.04 * whole.float().norm()
    assert cache.lengths.tolist() == [n] * 3
    with pytest.raises(ValueError, match="full"):
        layer.token(x[:, 0], positions[0].expand(3, 3), cache)
    with pytest.raises(ValueError, match="right"):
        ContextLayer(device=dev).token(x[:, 0], positions[0].expand(3, 3), cache)


@pytest.mark.parametrize("bits", [8, 32])
def test_training_learns(dev, bits):
    """From a loss of log 2 (the head starts at zeros) to less than two thirds of it in 60 steps, and no value lost."""
    losses = train(60, state_bits=bits, device=dev)
    print(f"losses {losses[0]:.3f} .. {losses[-1]:.3f}", flush=True)
    assert abs(losses[0] - math.log(2)) < 1e-3 and all(math.isfinite(x) for x in losses)
    assert sum(losses[-10:]) / 10 < 2 / 3 * math.log(2)
