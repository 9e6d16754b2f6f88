"""Forward-mode derivatives of the context layer's operators: refused, not dropped (CPU only: the refusal comes before
anything else that concerns a device)."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from rsna_knee_efficiency_amd import context

BF = torch.bfloat16


def _t(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


POS, LENGTHS = _t(4, 1, dtype=torch.int32), _t(1, dtype=torch.int32)
# a call and its tensors, every one of which may have a tangent
CALLS = {
    "layer_norm": (context.layer_norm, [_t(4, 8), _t(8), _t(8)]),
    "layer_norm_forward": (context.layer_norm_forward, [_t(4, 8), _t(8), _t(8)]),
    "layer_norm_backward": (context.layer_norm_backward, [_t(4, 8), _t(4, 8), _t(8), _t(4), _t(4)]),
    "rotary": (lambda x: context.rotary(x, POS, (8,)), [_t(1, 4, 2, 16)]),
    "rotary out": (lambda x: context.rotary(x, POS, (8,), out=x), [_t(1, 4, 2, 16)]),
    "rotary positions": (lambda p: context.rotary(_t(1, 4, 2, 16), p, (8,)), [_t(4, 1)]),
    "window_attention": (context.window_attention, [_t(1, 4, 2, 64, dtype=BF) for _ in range(3)]),
    "window_attention_forward": (context.window_attention_forward, [_t(1, 4, 2, 64, dtype=BF) for _ in range(3)]),
    "window_attention_backward": (context.window_attention_backward,
                                  [_t(1, 4, 2, 64, dtype=BF) for _ in range(5)] + [_t(1, 2, 4)]),
    "window_attention_token": (lambda q, k, v: context.window_attention_token(q, k, v, LENGTHS),
                               [_t(1, 2, 64, dtype=BF), _t(1, 9, 2, 64, dtype=BF), _t(1, 9, 2, 64, dtype=BF)]),
}


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("also_backward", [False, True])
def test_tangents_are_refused(name, also_backward):
    call, tensors = CALLS[name]
    for i in range(len(tensors)):
        args = [t.clone() for t in tensors]
        if also_backward:
            args = [t.requires_grad_() for t in args]
        with forward_ad.dual_level():
            args[i] = forward_ad.make_dual(args[i], torch.ones_like(args[i]))
            with pytest.raises(NotImplementedError, match="tangent"):
                call(*args)
    # inside a level, tensors without a tangent are taken as ever (and here refused for their device)
    with forward_ad.dual_level(), pytest.raises(ValueError, match="one GPU"):
        call(*[t.clone() for t in tensors])
