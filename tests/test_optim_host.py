"""What AdamW refuses before any launch (CPU only: an optimizer without its device memory, and no call reaches the
library)."""
from __future__ import annotations

import pytest
import torch

from rsna_knee_efficiency_amd import hip, optim


def _optimizer(monkeypatch, params, made_on="cuda:0"):
    """An optimizer whose parameters were on `made_on` when it was made; every launch it makes is kept in `launched`."""
    with monkeypatch.context() as m:
        m.setattr(optim.AdamW, "_check", lambda self, p: None)
        opt = optim.AdamW(params)
    opt.device = torch.device(made_on)
    opt.launched = []
    monkeypatch.setattr(torch.cuda, "current_device", lambda: opt.device.index)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(hip, "launch", lambda name, device, *args: opt.launched.append(args))
    return opt


def test_a_parameter_that_moved_to_the_host_is_refused(monkeypatch):
    p = torch.zeros((3, 4))
    opt = _optimizer(monkeypatch, [p])
    with pytest.raises(ValueError, match="parameter has changed"):
        opt.step([torch.zeros((3, 4))])
    assert opt.launched == [] and opt.step_count == 0


F32, BF16 = torch.float32, torch.bfloat16


def _run(opt, grads):
    """(step number, types, tensors) of every launch of a step"""
    opt.launched.clear()
    opt.device = torch.device("cpu")                        # (so that the tensors here are where they should be)
    with pytest.MonkeyPatch.context() as m:
        m.setattr(torch.cuda, "current_device", lambda: None)
        m.setattr(torch.Tensor, "get_device", lambda self: None)
        opt.step(grads)
    return [(a.step, (a.dtype, a.grad_dtype), a.count) for a, in opt.launched]


def test_every_tensor_counts_its_own_steps(monkeypatch):
    p = [torch.zeros(5), torch.zeros(3, dtype=BF16), torch.zeros(7), torch.zeros(2)]
    g = [torch.zeros_like(t) for t in p]
    opt = _optimizer(monkeypatch, p)
    assert _run(opt, g) == [(1, (0, 0), 3), (1, (1, 1), 1)]
    assert _run(opt, [g[0], None, None, g[3]]) == [(2, (0, 0), 2)]
    assert opt.steps == [2, 1, 1, 2] and opt.step_count == 2
    assert _run(opt, [None] * 4) == [] and opt.steps == [2, 1, 1, 2] and opt.step_count == 3
    state = opt.state_dict()
    assert _run(opt, g) == [(3, (0, 0), 2), (2, (1, 1), 1), (2, (0, 0), 1)]
    assert _run(opt, [None, g[1], g[2], None]) == [(3, (1, 1), 1), (3, (0, 0), 1)]
    assert _run(opt, g) == [(4, (0, 0), 3), (4, (1, 1), 1)] and opt.steps == [4] * 4
    opt.load_state_dict(state)
    assert opt.steps == [2, 1, 1, 2] and opt.step_count == 3
    opt.load_state_dict({n: t for n, t in state.items() if n != "steps"})
    assert opt.steps == [3] * 4
    for bad in ({"steps": [1]}, {"steps": [1, 1, -1, 1]}, {"step": -1}):
        with pytest.raises(ValueError, match="step"):
            opt.load_state_dict(state | bad)
    assert opt.steps == [3] * 4


def test_parameters_that_share_memory_are_refused(monkeypatch):
    flat = torch.zeros(100)
    for pair in ((flat[:50], flat[49:]), (flat, flat.view(10, 10)), (flat[20:30], flat)):
        with pytest.raises(ValueError, match="share memory"):
            _optimizer(monkeypatch, list(pair))
    _optimizer(monkeypatch, [flat[50:], flat[:50], torch.zeros(0), torch.zeros(0), torch.zeros(3)])
