"""The sums of attention weight that the cache manager keeps beside the keys (no GPU)."""

import math

import pytest
import torch

from simple_inference_amd.cache import CacheManager
from simple_inference_amd.parts.model import CacheLayout
from simple_inference_amd.parts.plan import PagedKVNeed


def manager(needs=(PagedKVNeed(2, 8, None),), slabs=(3,), runs=((0, 0), (0, 2), None, (0, 1))):
    plan = CacheLayout(kv_groups=list(needs), kv_slabs=list(slabs), run_kv=list(runs), states=[], run_state=[None] * len(runs))
    return CacheManager(plan, page_size=4, num_pages=12, max_running=3, dtype=torch.float32, device="cpu")


def test_layers_have_their_sums():
    cache = manager()
    assert all(c.weights is None for c in cache.layer_caches([torch.zeros(1, 1, dtype=torch.int32)]))
    cache.keep_weights(40)
    layers = cache.layer_caches([torch.zeros(1, 1, dtype=torch.int32)])
    for c in layers:
        if c.k_pages is None:
            assert c.weights is None
            continue
        assert c.weights.shape == (4, 2, 40) and c.weights.dtype == torch.float32 and c.weights.is_contiguous() and not c.weights.any()
    layers[0].weights.fill_(1.0)
    assert not layers[1].weights.any() and not layers[3].weights.any()


def test_groups_have_sums_of_their_own():
    cache = manager((PagedKVNeed(2, 8, None), PagedKVNeed(1, 16, 8)), (1, 2), ((0, 0), (1, 1), (1, 0)))
    cache.keep_weights(16)
    shapes = [tuple(c.weights.shape) for c in cache.layer_caches([torch.zeros(1, 1, dtype=torch.int32)] * 2)]
    assert shapes == [(4, 2, 16), (4, 1, 16), (4, 1, 16)]


def test_sums_of_adopted_places_begin_at_zero():
    cache = manager()
    cache.keep_weights(40)
    weights = cache.groups[0].weights
    cache.admit(1, 20, 4)
    cache.extend(1, 14)
    weights.fill_(math.nan)                      # what earlier requests left in every row
    slot = cache.admit(2, 20, 4, shared_pages=cache.table(0, 1)[:2])
    assert cache.lengths[2] == 8
    assert not weights[:, slot, :, :8].any() and weights[:, slot, :, 8:].isnan().all()
    assert all(weights[:, other].isnan().all() for other in range(4) if other != slot)
    plain = cache.admit(3, 4, 4)                 # its own first step begins its sums
    assert weights[:, plain].isnan().all()


def test_keep_weights_refuses():
    cache = manager()
    for places in (0, -4):
        with pytest.raises(ValueError):
            cache.keep_weights(places)
    cache.admit(1, 8, 4)
    with pytest.raises(ValueError):
        cache.keep_weights(40)
