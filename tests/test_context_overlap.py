"""Where rotary's output may lie (CPU only: what the library is called with; no kernel runs)."""
from __future__ import annotations

import random

import pytest
import torch

from rsna_knee_efficiency_amd import context, hip

POS = torch.zeros((6, 1), dtype=torch.int32)


@pytest.fixture
def calls(monkeypatch):
    """The tensors' addresses of every call that reaches the library"""
    seen = []
    monkeypatch.setattr(context, "_on_gpu", lambda *t: None)
    monkeypatch.setattr(hip, "launch", lambda name, device, a: seen.append((a.x, a.y)))
    return seen


def _elements(t):
    at = torch.zeros(t.shape, dtype=torch.int64)
    for d, (n, s) in enumerate(zip(t.shape, t.stride())):
        at = at + (torch.arange(n) * s).view(-1, *[1] * (t.dim() - 1 - d))
    return set((at + t.storage_offset()).flatten().tolist())


def test_elements_in_common_are_found():
    """Views of one buffer at random offsets: never denied, and exact where strides are the same and nested."""
    rng = random.Random(1)
    buf = torch.zeros(5000)
    exact = 0
    for _ in range(3000):
        shape = [rng.randint(1, 3), rng.randint(1, 6), rng.randint(1, 4), rng.choice([2, 4, 8])]
        inner = shape[3] + rng.choice([0, 0, 3, 8])
        strides = [0, inner * shape[2] + rng.choice([0, 0, 5, 40]), inner, 1]
        strides[0] = strides[1] * shape[1] + rng.choice([0, 7])
        if rng.random() < 0.3:
            strides[1], strides[2] = inner, inner * shape[1]
            strides[0] = inner * shape[1] * shape[2]
        other = list(strides) if rng.random() < 0.7 else [strides[1], strides[0], strides[2], 1]
        x = buf.as_strided(shape, strides, rng.randint(0, 300))
        y = buf.as_strided(shape, other, rng.randint(0, 300))
        common = bool(_elements(x) & _elements(y))
        got = context._may_meet(x, y)
        assert got or not common, (shape, strides, other)
        if strides == other:
            assert got == common, (shape, strides, x.storage_offset(), y.storage_offset())
            exact += common
    assert 100 < exact < 2900
    far = torch.zeros(100).view(1, 5, 2, 10)
    assert not context._may_meet(buf[:100].view(1, 5, 2, 10), far)
    slides = buf.as_strided((1, 200, 1, 64), (0, 1, 0, 1))         # every row meets the next ones
    assert context._may_meet(slides, buf.as_strided((1, 200, 1, 64), (0, 1, 0, 1), 5))


def test_out_beside_and_across_x(calls):
    packed = torch.zeros((1, 6, 3, 4, 16))
    for x, out, copied in [(packed[:, :, 0], packed[:, :, 0], False),       # in place
                           (packed[:, :, 0], packed[:, :, 2], False),       # beside each other
                           (packed[:, :, 0], packed[:, :, 0, :, :].clone(), False),
                           (packed.flatten(2, 3)[:, :, :8], packed.flatten(2, 3)[:, :, 2:10], True),
                           (packed.flatten(2, 3)[:, :, 2:10], packed.flatten(2, 3)[:, :, :8], True),
                           (packed.view(1, 6, 12, 16)[:, :, ::2], packed.view(1, 6, 12, 16)[:, :, 1::2], False)]:
        context.rotary(x, POS, (8,), out=out)
        at, to = calls.pop()
        assert to == out.data_ptr() and (at != x.data_ptr()) == copied
    shifted = torch.zeros((1, 7, 4, 16))
    context.rotary(shifted[:, :6], POS, (8,), out=shifted[:, 1:])
    assert calls.pop()[0] != shifted.data_ptr()


def test_expanded_out_is_refused(calls):
    one = torch.zeros((1, 6, 1, 16)).expand(-1, -1, 4, -1)
    for x, out in ((one, one), (torch.zeros((1, 6, 4, 16)), one)):
        with pytest.raises(ValueError, match="one place"):
            context.rotary(x, POS, (8,), out=out)
    context.rotary(one, POS, (8,))             # read, an expanded tensor is as good as any
    assert len(calls) == 1
