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


LR, B1, B2, EPS, WD = 3e-3, 0.9, 0.99, 1e-8, 0.02


@pytest.mark.parametrize("bits", [32, 8])
def test_a_first_gradient_that_comes_late(dev, bits):
    """Tensors left out of some steps, the first until the eleventh: each follows the formula in float64 with its own
    step number, the others' moments do not enter.  Float32 is off by 2^-24 of each result, about 16 of them in a step
    whose update is below 20 lr (see sqrt(v) beside eps); 8-bit moments begin at zeros, so the first step is
    float32's."""
    g = torch.Generator(device=dev).manual_seed(1)
    params = [torch.randn(n, generator=g, device=dev) for n in (300, 1000, 40, 7)]
    want = [p.double() for p in params]
    m, v, t = [torch.zeros_like(p) for p in want], [torch.zeros_like(p) for p in want], [0] * 4
    opt = optim.AdamW(params, LR, (B1, B2), EPS, WD, bits)
    for step in range(12):
        takes = [step >= 10, True, step % 3 == 0, step in (0, 11)]
        grads = [torch.randn(p.shape, generator=g, device=dev) * 0.1 if on else None for p, on in zip(params, takes)]
        opt.step(grads)
        for i, x in enumerate(grads):
            if x is None:
                continue
            t[i] += 1
            m[i], v[i] = B1 * m[i] + (1 - B1) * x.double(), B2 * v[i] + (1 - B2) * x.double() ** 2
            want[i] = want[i] * (1 - LR * WD) - LR * (m[i] / (1 - B1 ** t[i])) / ((v[i] / (1 - B2 ** t[i])).sqrt() + EPS)
            if bits == 32 or t[i] == 1:
                off = (params[i].double() - want[i]).abs()
                assert (off <= 2.0 ** -24 * (4 * t[i] * want[i].abs() + 32 * t[i] * LR * 20)).all(), (step, i)
    assert opt.steps == t == [2, 12, 4, 2] and opt.step_count == 12


def test_a_constant_gradient_moves_by_the_rate(dev):
    """m / (1 - beta1^t) and v / (1 - beta2^t) of a constant gradient are itself and its square at every t of its own:
    a step moves by lr, after a thousand steps of another tensor too (a dozen float32 roundings: below 1e-5 of it)."""
    late, other = (torch.zeros(64, device=dev) for _ in range(2))
    one = torch.ones(64, device=dev)
    opt = optim.AdamW([late, other], lr=1e-3, betas=(0.9, 0.999), weight_decay=0.0)
    for _ in range(1000):
        opt.step([None, one])
    for t in range(1, 6):
        opt.step([one, one])
        assert ((late + t * 1e-3).abs() <= t * 1e-3 * 1e-5).all()


def test_step_numbers_travel(dev):
    g = torch.Generator(device=dev).manual_seed(2)
    a = [torch.randn(n, generator=g, device=dev) for n in (300, 20)]
    x = [torch.randn(n, generator=g, device=dev) for n in (300, 20)]
    one = optim.AdamW(a, LR, (B1, B2), EPS, WD, 8)
    for _ in range(3):
        one.step([x[0], None])
    b = [t.clone() for t in a]
    two = optim.AdamW(b, LR, (B1, B2), EPS, WD, 8)
    two.load_state_dict(one.state_dict())
    one.step(x)
    two.step(x)
    assert two.steps == one.steps == [4, 1] and all(torch.equal(s, t) for s, t in zip(a, b))
