"""A context layer over all the tokens of a study, from the operators of `context` and `optim`: in training, over whole
studies, and for tokens that arrive one at a time.

The reference's context layer (src/knee/models/baseline.py:954-977) is one pre-norm transformer layer over a study's
window features.  This is the same layer over every position of the encoder's last map: its tokens lie at a slice, a
row and a column (rotary positions in place of a learned table), see the tokens within a window and a few first
summary tokens, and absent series are masked.

    python rsna-knee-efficiency_amd/context_layer.py --steps 60        # trains one on synthetic studies
"""
from __future__ import annotations

import argparse
import math

import torch
import torch.nn.functional as F

if __package__ in (None, ""):                  # run as a file
    import sys
    from pathlib import Path
    sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
    import __graft_entry__
    __graft_entry__.load_package()
    from rsna_knee_efficiency_amd import context, optim
else:
    from . import context, optim

HEAD_DIM = 64                                  # channels a head, as in the reference's context layer


def study_positions(slices: int, rows: int, cols: int, summary: int, device) -> torch.Tensor:
    """(summary + slices * rows * cols, 3) int32: slice, row and column of a study's tokens, slice by slice; the summary
    tokens before them lie at the origin."""
    grid = torch.stack(torch.meshgrid(*(torch.arange(n) for n in (slices, rows, cols)), indexing="ij"), -1)
    return torch.cat([torch.zeros((summary, 3), dtype=torch.int64), grid.reshape(-1, 3)]).to(device, torch.int32)


class TokenCache:
    """Keys and values of the tokens that have arrived, and how many of each row."""

    def __init__(self, layer: "ContextLayer", batch: int, capacity: int) -> None:
        shape = (batch, capacity, layer.key_heads, HEAD_DIM)
        self.k, self.v = (torch.zeros(shape, dtype=layer.dtype, device=layer.device) for _ in range(2))
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=layer.device)
        self.arrived = 0                       # tokens appended: every row's length, known to the host


class ContextLayer:
    """One pre-norm transformer layer of `width` channels.  Weights are float32 (`params`, for an optimizer); activations
    and products are of `dtype`.  left, right, sinks: the window of `context.window_attention`; sections: pairs of
    channels that turn with slice, row and column."""

    def __init__(self, width: int = 256, heads: int = 4, key_heads: int | None = None, ff: int = 512, left: int | None = 512,
                 right: int | None = 512, sinks: int = 12, sections=(8, 12, 12), dtype=torch.bfloat16, device="cuda:0",
                 seed: int = 0) -> None:
        self.heads, self.key_heads = heads, heads if key_heads is None else key_heads
        if heads % self.key_heads:
            raise ValueError("heads must be a multiple of key_heads")
        self.width, self.left, self.right, self.sinks, self.sections = width, left, right, sinks, tuple(sections)
        self.dtype, self.device = dtype, torch.device(device)
        g = torch.Generator().manual_seed(seed)
        inner = heads * HEAD_DIM

        def weight(out: int, into: int) -> torch.Tensor:
            return torch.randn((out, into), generator=g) / math.sqrt(into)
        made = {"ln1_w": torch.ones(width), "ln1_b": torch.zeros(width),
                "qkv_w": weight((heads + 2 * self.key_heads) * HEAD_DIM, width), "qkv_b": torch.zeros((heads + 2 * self.key_heads) * HEAD_DIM),
                "out_w": weight(width, inner), "out_b": torch.zeros(width),
                "ln2_w": torch.ones(width), "ln2_b": torch.zeros(width),
                "ff1_w": weight(ff, width), "ff1_b": torch.zeros(ff), "ff2_w": weight(width, ff), "ff2_b": torch.zeros(width)}
        self.w = {n: t.to(self.device).requires_grad_() for n, t in made.items()}

    @property
    def params(self) -> list[torch.Tensor]:
        return list(self.w.values())

    def _linear(self, x: torch.Tensor, name: str) -> torch.Tensor:
        rows = F.linear(x.reshape(-1, x.shape[-1]), self.w[name + "_w"].to(x.dtype), self.w[name + "_b"].to(x.dtype))
        return rows.view(*x.shape[:-1], -1)

    def _project(self, x: torch.Tensor, positions: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """(q, k, v) (batch, tokens, heads, channels): queries and keys turned by their positions in one call"""
        h = self._linear(context.layer_norm(x, self.w["ln1_w"], self.w["ln1_b"]), "qkv")
        h = h.view(*x.shape[:2], self.heads + 2 * self.key_heads, HEAD_DIM)
        turned = context.rotary(h[:, :, :self.heads + self.key_heads], positions, self.sections)
        return turned[:, :, :self.heads], turned[:, :, self.heads:], h[:, :, self.heads + self.key_heads:]

    def _rest(self, x: torch.Tensor, attended: torch.Tensor) -> torch.Tensor:
        x = x + self._linear(attended.flatten(2), "out")
        h = context.layer_norm(x, self.w["ln2_w"], self.w["ln2_b"])
        return x + self._linear(torch.relu(self._linear(h, "ff1")), "ff2")

    def __call__(self, x: torch.Tensor, positions: torch.Tensor, key_mask: torch.Tensor | None = None) -> torch.Tensor:
        """x (batch, tokens, width), positions (tokens, 3) or (batch, tokens, 3), key_mask (batch, tokens) -> like x.
        Differentiable in x and the weights."""
        x = x.to(self.dtype)
        q, k, v = self._project(x, positions)
        return self._rest(x, context.window_attention(q, k, v, self.left, self.right, self.sinks, key_mask))

    @torch.no_grad()
    def token(self, x: torch.Tensor, positions: torch.Tensor, cache: TokenCache) -> torch.Tensor:
        """One new token a row: x (batch, width), positions (batch, 3) -> (batch, width), its keys and values appended to
        the cache.  The layer sees no later tokens (right = 0)."""
        if self.right != 0:
            raise ValueError("tokens one at a time need a layer with right = 0")
        if cache.arrived >= cache.k.shape[1]:
            raise ValueError("the cache is full")
        if x.shape != (cache.k.shape[0], self.width):
            raise ValueError("x must be (the cache's batch, width)")
        x = x.to(self.dtype)[:, None]
        q, k, v = self._project(x, positions[:, None])
        cache.k[:, cache.arrived], cache.v[:, cache.arrived] = k[:, 0], v[:, 0]
        cache.arrived += 1
        cache.lengths += 1
        out = context.window_attention_token(q[:, 0], cache.k, cache.v, cache.lengths, self.left, self.sinks)
        return self._rest(x, out[:, None])[:, 0]


def train(steps: int = 60, studies: int = 4, slices: int = 8, side: int = 9, findings: int = 12, state_bits: int = 8,
          seed: int = 0, device="cuda:0") -> list[float]:
    """Trains a layer and a linear head on synthetic studies: the tokens of a study are noise, a finding's direction is
    added to a few of them, and the head reads the findings from the summary tokens, which see a first token's window
    only through the layer.  One slot in eight is absent.  -> the loss of every step."""
    summary = findings
    layer = ContextLayer(left=None, right=None, sinks=summary, device=device, seed=seed)
    g = torch.Generator(device=device).manual_seed(seed)
    positions = study_positions(slices, side, side, summary, device)
    n = positions.shape[0]
    directions = torch.randn((findings, layer.width), generator=g, device=device)
    start = torch.randn((summary, layer.width), generator=g, device=device).requires_grad_()
    head = torch.zeros(layer.width, device=device, requires_grad=True)
    params = [*layer.params, start, head]
    opt = optim.AdamW(params, lr=2e-3, weight_decay=1e-4, state_bits=state_bits)
    losses = []
    for _ in range(steps):
        there = torch.rand((studies, findings), generator=g, device=device) < 0.5
        x = torch.randn((studies, n - summary, layer.width), generator=g, device=device)
        mask = torch.ones((studies, n), dtype=torch.bool, device=device)
        mask[:, summary:] = (torch.rand((studies, 8), generator=g, device=device) > 0.125).repeat_interleave(-(-(n - summary) // 8), 1)[:, :n - summary]
        at = torch.rand((studies, findings, n - summary), generator=g, device=device).masked_fill(~mask[:, None, summary:], -1.0)
        where = at.topk(6, -1).indices                     # six tokens of present slots show a finding
        shown = (there[:, :, None] * 1.0).expand(-1, -1, 6)
        for f in range(findings):
            x.scatter_add_(1, where[:, f, :, None].expand(-1, -1, layer.width), shown[:, f, :, None] * directions[f])
        tokens = torch.cat([start.expand(studies, -1, -1), x], 1)
        out = layer(tokens, positions, mask)
        logits = (out[:, :summary].float() * head).sum(-1)
        loss = F.binary_cross_entropy_with_logits(logits, there.float())
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.detach())
    return torch.stack(losses).tolist()


def main() -> None:
    ap = argparse.ArgumentParser(description="Trains a context layer on synthetic studies.")
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--studies", type=int, default=4)
    ap.add_argument("--state-bits", type=int, default=8, choices=(8, 32))
    a = ap.parse_args()
    losses = train(a.steps, a.studies, state_bits=a.state_bits)
    for i in range(0, len(losses), max(1, len(losses) // 10)):
        print(f"step {i:4d}  loss {losses[i]:.4f}")
    print(f"last ten {sum(losses[-10:]) / len(losses[-10:]):.4f}")


if __name__ == "__main__":
    main()
