"""The books of a cache whose requests have dropped some of their tokens (no GPU)."""

import pytest

from simple_inference_amd.cache import CacheManager
from simple_inference_amd.parts.model import CacheLayout
from simple_inference_amd.parts.plan import PagedKVNeed


def manager(num_pages=12, page_size=4, needs=(PagedKVNeed(2, 8, None),)):
    layout = CacheLayout(kv_groups=list(needs), kv_slabs=[1] * len(needs), run_kv=[(g, 0) for g in range(len(needs))],
                         states=[], run_state=[None] * len(needs))
    import torch
    return CacheManager(layout, page_size=page_size, num_pages=num_pages, max_running=3, dtype=torch.float32, device="cpu",
                        allocate_storage=False)


@pytest.mark.parametrize("reserved", [True, False])
def test_shrink_gives_pages_back_and_goes_on(reserved):
    cache = manager()
    cache.admit(5, 40 if reserved else None, 16)
    cache.extend(5, 33)
    assert len(cache.table(0, 5)) == 9 and cache.owns_pages(5)
    before, first = cache.free_pages(), list(cache.table(0, 5))
    version = cache.groups[0].versions[5]
    cache.shrink(5, 13)
    cache.check()
    assert cache.lengths[5] == 13 and cache.table(0, 5) == first[:4] and cache.free_pages() == before + 5
    assert cache.groups[0].versions[5] != version
    assert cache.groups[0].pool.n_promised >= 5                # nobody else can take what the request may need again
    for n in range(20):                                        # as many tokens again, cut back on the way
        assert cache.extend(5, 1) == cache.lengths[5] - 1
        if cache.lengths[5] > 16:
            cache.shrink(5, 13)
    cache.check()
    cache.shrink(5, cache.lengths[5])                          # nothing to give back
    cache.release(5)
    assert cache.free_pages() == 12


def test_shrink_within_a_page_keeps_the_table():
    cache = manager()
    cache.admit(1, 12, 4)
    cache.extend(1, 11)
    version = cache.groups[0].versions[1]
    cache.shrink(1, 9)
    assert cache.lengths[1] == 9 and len(cache.table(0, 1)) == 3 and cache.groups[0].versions[1] == version


def test_shrink_refuses():
    cache = manager()
    cache.admit(1, 12, 4)
    cache.extend(1, 8)
    for tokens in (0, -1, 9):
        with pytest.raises(ValueError):
            cache.shrink(1, tokens)
    cache.admit(2, 12, 4, shared_pages=cache.table(0, 1)[:1])
    assert not cache.owns_pages(1) and not cache.owns_pages(2)
    for req, tokens in ((1, 4), (2, 2)):
        with pytest.raises(ValueError):
            cache.shrink(req, tokens)
    cache.release(2)
    cache.groups[0].pool.pin(cache.table(0, 1)[0])             # a prefix that is kept for others
    with pytest.raises(ValueError):
        cache.shrink(1, 4)
    assert cache.lengths[1] == 8
    cache.check()
    windowed = manager(needs=(PagedKVNeed(2, 8, None), PagedKVNeed(2, 8, 16)))
    windowed.admit(1, 12, 4)
    windowed.extend(1, 8)
    with pytest.raises(ValueError):
        windowed.shrink(1, 4)
