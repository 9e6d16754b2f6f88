"""A context layer's cache: a call that is refused leaves it as it was."""
from __future__ import annotations

import pytest
import torch

from rsna_knee_efficiency_amd.context_layer import ContextLayer, TokenCache

pytestmark = pytest.mark.gpu


def test_a_refused_token_leaves_the_cache(dev):
    layer = ContextLayer(heads=2, key_heads=1, left=50, right=0, sinks=2, device=dev)
    cache = TokenCache(layer, 3, 5)
    x, at = torch.randn((3, 256), device=dev), torch.zeros((3, 3), dtype=torch.int32, device=dev)
    layer.token(x, at, cache)
    kept = cache.k.clone(), cache.v.clone()
    for bad in ((x[:1], at[:1]), (x[:, :200], at), (x, at[:, :2]), (torch.cat([x, x]), torch.cat([at, at]))):
        with pytest.raises((ValueError, RuntimeError)):
            layer.token(*bad, cache)
        assert cache.arrived == 1 and cache.lengths.tolist() == [1] * 3
        assert torch.equal(cache.k, kept[0]) and torch.equal(cache.v, kept[1])
    layer.token(x, at, cache)
    assert cache.arrived == 2
