"""AdamW over many tensors at once on the GPU (`d8s_adamw`, include/d8s_hip.h): the optimizer that trains a head or a
context layer, with moments in 32 or 8 bits.

    opt = AdamW(model.parameters(), lr=1e-3, state_bits=8)
    loss.backward()
    opt.step()                           # or opt.step(grads), opt.step(grad_scale=scale on the GPU)

A step is one launch for every 100 tensors of one pair of types (and, where some were left out of earlier steps, of one
step number), whatever their sizes.  There is no CPU path: without
the library the calls raise.
"""
from __future__ import annotations

import numpy as np
import torch

from . import hip

_ROW = np.dtype([("p", "u8"), ("g", "u8"), ("n", "i8"), ("at", "i8")])       # AdamwTensor


class AdamW:
    """p = p (1 - lr weight_decay) - lr / (1 - beta1^t) m / (sqrt(v) / sqrt(1 - beta2^t) + eps) after
    m = beta1 m + (1 - beta1) g and v = beta2 v + (1 - beta2) g^2, all in float32 with every operation rounded by
    itself, p then to its type.  t counts a tensor's own steps (`steps`): one that is left out of a step keeps its
    number with its moments.

    params: contiguous float32, bfloat16 or float16 tensors on one GPU; gradients are float32 or 16 bits beside
    float32 parameters, float32 or the parameter's own type beside 16-bit ones.  The moments of all tensors lie in
    one array each, tensor i's padded to whole blocks of 256 elements (the padding stays zeros).  state_bits 8 keeps
    them as codes with one float32 scale a block, 2.03 bytes an element in place of 8: m = scale c |c| / 127^2 and
    sqrt(v) = scale c^2 / 255^2.  Gradients must be finite: one that is not spoils its element, with state_bits 8
    its block's moments."""

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.01,
                 state_bits: int = 32) -> None:
        self.params = list(params)
        if not self.params:
            raise ValueError("no parameters")
        if state_bits not in (8, 32):
            raise ValueError("state_bits must be 8 or 32")
        if len({id(p) for p in self.params}) != len(self.params):
            raise ValueError("a parameter is given twice")
        if not (lr >= 0 and eps > 0 and weight_decay >= 0 and 0 <= betas[0] < 1 and 0 <= betas[1] < 1):
            raise ValueError("lr and weight_decay must not be negative, eps positive, betas in [0, 1)")
        self.device = self.params[0].device
        for p in self.params:
            self._check(p)
        spans = sorted((p.data_ptr(), p.numel() * p.element_size()) for p in self.params if p.numel())
        if any(at + size > after for (at, size), (after, _) in zip(spans, spans[1:])):
            raise ValueError("parameters share memory")      # (two updates of one element would run at once)
        self.lr, self.betas, self.eps, self.weight_decay, self.state_bits = lr, tuple(betas), eps, weight_decay, state_bits
        self.step_count = 0                    # calls of `step`
        # the number of steps of every tensor: one for all as long as none is left out of one, else a list
        self._steps: int | list[int] = 0
        block = hip.ADAMW_BLOCK
        self._table = np.zeros(len(self.params), _ROW)
        self._table["n"] = [p.numel() for p in self.params]
        padded = (self._table["n"] + block - 1) // block * block
        self._table["at"] = np.cumsum(padded) - padded
        total = max(block, int(padded.sum()))

        def zeros(n, dtype):
            return torch.zeros(n, dtype=dtype, device=self.device)
        if state_bits == 8:
            self._state = {"m_code": zeros(total, torch.int8), "v_code": zeros(total, torch.uint8),
                           "m_scale": zeros(total // block, torch.float32), "v_scale": zeros(total // block, torch.float32)}
        else:
            self._state = {"m": zeros(total, torch.float32), "v": zeros(total, torch.float32)}
        # what a step checks its tensors against
        self._shapes, self._dtypes = [p.shape for p in self.params], [p.dtype for p in self.params]

    def _check(self, p: torch.Tensor) -> None:
        if p.dtype not in hip.ELEMENTS or not p.is_contiguous() or p.device != self.device or p.device.type != "cuda":
            raise ValueError("parameters must be contiguous float32, bfloat16 or float16 tensors on one GPU")

    @property
    def steps(self) -> list[int]:
        """How many steps each tensor has taken."""
        return [self._steps] * len(self.params) if isinstance(self._steps, int) else list(self._steps)

    def step(self, grads=None, grad_scale: torch.Tensor | None = None) -> None:
        """One step in place.  grads: a tensor, or None, for every parameter (default: their .grad); parameters
        without one are left as they are, their moments and their number of steps too.  grad_scale: one float32 on the GPU that every
        gradient is multiplied by.  The step's numbers are arguments of its launches, so it cannot be recorded into
        a graph."""
        grads = [p.grad for p in self.params] if grads is None else list(grads)
        if len(grads) != len(self.params):
            raise ValueError("a gradient (or None) for every parameter is required")
        if torch.cuda.current_device() != self.device.index:
            with torch.cuda.device(self.device):
                return self._step(grads, grad_scale)
        return self._step(grads, grad_scale)

    def _step(self, grads: list, grad_scale: torch.Tensor | None) -> None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("an optimizer step cannot be recorded into a graph")
        if grad_scale is not None and (grad_scale.numel() != 1 or grad_scale.dtype != torch.float32
                                       or grad_scale.device != self.device):
            raise ValueError("grad_scale must be one float32 on the parameters' GPU")
        params, shapes, dtypes, table, which = self.params, self._shapes, self._dtypes, self._table, None
        if any(g is None for g in grads):
            which = [i for i, g in enumerate(grads) if g is not None]
            params, grads, shapes, dtypes = ([x[i] for i in which] for x in (params, grads, shapes, dtypes))
            table = table[which]
        on = self.device.index                 # (the kernel follows raw pointers: a moved parameter's is another device's)
        if ([p.shape for p in params] != shapes or [p.dtype for p in params] != dtypes
                or not all(p.get_device() == on and p.is_contiguous() for p in params)):
            raise ValueError("a parameter has changed its shape, type, layout or device")
        if [g.shape for g in grads] != shapes or any(g.get_device() != on for g in grads):
            raise ValueError("a gradient must have its parameter's shape and device")
        kinds = list(zip(dtypes, [g.dtype for g in grads]))
        for pt, gt in set(kinds):
            if gt not in hip.ELEMENTS or not (gt == pt or torch.float32 in (gt, pt)):
                raise ValueError(f"a gradient of {gt} beside a parameter of {pt}")
        grads = [g if g.is_contiguous() else g.contiguous() for g in grads]     # (held until the launches are made)
        table["p"], table["g"] = [p.data_ptr() for p in params], [g.data_ptr() for g in grads]
        s = self._state
        at = [t.data_ptr() for t in s.values()] + [0] * (4 - len(s))
        if which is None and isinstance(self._steps, int):
            numbers, after = [self._steps + 1], self._steps + 1
            groups = kinds
        else:
            after = self.steps
            for i in range(len(after)) if which is None else which:
                after[i] += 1
            numbers = after if which is None else [after[i] for i in which]
            groups = list(zip(kinds, numbers))
            after = after[0] if len(set(after)) == 1 else after
        for group in dict.fromkeys(groups):
            rows = table if groups.count(group) == len(groups) else table[[i for i, x in enumerate(groups) if x == group]]
            (pt, gt), number = (group, numbers[0]) if groups is kinds else group
            hip.launch("d8s_adamw", self.device, hip.AdamwArgs(
                rows.ctypes.data, *at, 0 if grad_scale is None else grad_scale.data_ptr(), number, self.lr,
                *self.betas, self.eps, self.weight_decay, len(rows), hip.ELEMENTS[pt], hip.ELEMENTS[gt],
                self.state_bits))
        self.step_count += 1
        self._steps = after
        torch.autograd.graph.increment_version([*params, *s.values()])

    def moments(self) -> tuple[torch.Tensor, torch.Tensor]:
        """Both moments of all tensors, (elements,) float32, laid out as the state is: the state's own arrays, or
        new ones of the values that 8-bit moments stand for."""
        s = self._state
        if self.state_bits == 32:
            return s["m"], s["v"]
        m, v = (torch.empty(s["m_code"].numel(), dtype=torch.float32, device=self.device) for _ in range(2))
        hip.launch("d8s_adamw_moments", self.device, *(t.data_ptr() for t in s.values()), m.numel(), m.data_ptr(),
                   v.data_ptr())
        return m, v

    def zero_grad(self) -> None:
        for p in self.params:
            p.grad = None

    def state_dict(self) -> dict:
        """The step counts, of calls and of every tensor, and copies of the moments as they are kept."""
        return {"step": self.step_count, "steps": self.steps, **{n: t.clone() for n, t in self._state.items()}}

    def load_state_dict(self, state: dict) -> None:
        """Takes over what `state_dict` gave of an optimizer over tensors of the same sizes and state_bits.  Without
        "steps" every tensor has taken "step" of them."""
        if set(state) - {"steps"} != {"step", *self._state}:
            raise ValueError(f"the state must hold step, steps and {sorted(self._state)}")
        for n, t in self._state.items():
            if state[n].shape != t.shape or state[n].dtype != t.dtype:
                raise ValueError(f"{n} must be {tuple(t.shape)} {t.dtype}")
        step = int(state["step"])
        steps = [int(t) for t in state["steps"]] if "steps" in state else [step] * len(self.params)
        if step < 0 or any(t < 0 for t in steps):
            raise ValueError("step must not be negative")
        if len(steps) != len(self.params):
            raise ValueError("steps must hold a number for every parameter")
        for n, t in self._state.items():
            t.copy_(state[n])
        self.step_count, self._steps = step, steps[0] if len(set(steps)) == 1 else steps
