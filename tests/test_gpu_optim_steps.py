"""AdamW over the life of its parameters on the GPU: moved away and back, left out of some steps."""
from __future__ import annotations

import pytest
import torch

from rsna_knee_efficiency_amd import optim

pytestmark = pytest.mark.gpu


def test_a_moved_parameter_is_refused(dev):
    """`module.cpu()` replaces a parameter's data in place; the step raises and changes nothing until it is back."""
    layer = torch.nn.Linear(40, 30).to(dev)
    opt = optim.AdamW(layer.parameters())
    grads = [torch.ones_like(p) for p in layer.parameters()]
    opt.step(grads)
    layer.cpu()
    before = [p.detach().clone() for p in layer.parameters()]
    with pytest.raises(ValueError, match="parameter has changed"):
        opt.step(grads)
    assert opt.step_count == 1 and all(torch.equal(a, b) for a, b in zip(before, layer.parameters()))
    layer.to(dev)
    opt.step(grads)
    assert opt.step_count == 2 and not any(torch.equal(a.to(dev), b) for a, b in zip(before, layer.parameters()))
