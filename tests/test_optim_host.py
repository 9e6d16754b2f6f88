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
