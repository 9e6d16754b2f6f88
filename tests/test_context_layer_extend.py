"""A call of the context layer over its 8-bit cache that is refused leaves the cache as it was (CPU only, no kernel launches)."""
from __future__ import annotations

import pytest
import torch

from rsna_knee_efficiency_amd import context_layer, token_cache


@pytest.mark.parametrize("entry,how", [
    *[("extend", how) for how in (dict(left=-1), dict(sinks=-3), dict(right=-1), dict(heads=1 << 25), dict(counts=torch.zeros(2)))],
    *[("token", how) for how in (dict(left=-1), dict(sinks=-3), dict(heads=1 << 25))],
])
def test_a_refused_call_appends_nothing(entry, how, monkeypatch):
    layer = object.__new__(context_layer.ContextLayer)
    heads = how.get("heads", 4)
    layer.__dict__.update(width=256, heads=heads, key_heads=1, dtype=torch.bfloat16, left=how.get("left", 10), right=how.get("right", 0),
                          sinks=how.get("sinks", 0))
    cache = object.__new__(token_cache.QuantizedCache)
    cache.__dict__.update(batch=4, capacity=100, key_heads=1, channels=64, codes=torch.int8, dtype=torch.bfloat16,
                          _lengths=torch.zeros(4, dtype=torch.int32), device=torch.device("cuda:0"))
    monkeypatch.setattr(token_cache, "_on_gpu", lambda *t: None)
    monkeypatch.setattr(token_cache.QuantizedCache, "append", lambda *a: pytest.fail("the tokens were appended"))
    one = torch.zeros((1, 1, 1, 1), dtype=torch.bfloat16)
    monkeypatch.setattr(layer, "_project", lambda x, p: tuple(one.expand(4, x.shape[1], h, 64) for h in (heads, 1, 1)), raising=False)
    x, positions = torch.zeros((4, 3, 256)), torch.zeros((4, 3, 3))
    with pytest.raises(ValueError, match="left|right|sinks|too many|counts"):
        if entry == "token":
            layer.token(x[:, 0], positions[:, 0], cache)
        else:
            layer.extend(x, positions, cache, how.get("counts"))
