"""What an eviction gives back to the pool, and to whom (no GPU)."""

import pytest

from simple_inference_amd.cache.allocator import OutOfPages, PagePool
from test_cache_shrink import manager


@pytest.mark.parametrize("reserved", [True, False])
def test_pages_beyond_the_most_are_anybodys(reserved):
    cache = manager()
    cache.admit(1, 48 if reserved else None, 16)
    cache.extend(1, 48)                                    # all twelve pages
    assert not cache.can_admit(4)
    cache.shrink(1, 8, most=12)
    cache.check()
    pool = cache.groups[0].pool
    assert (len(cache.table(0, 1)), pool.n_free, pool.n_promised, pool.n_unpromised) == (2, 10, 1, 9)
    cache.admit(2, 36, 4)                                  # nine pages for another
    assert pool.n_unpromised == 0
    cache.extend(2, 36)
    for _ in range(3):                                     # the first grows to its most and is cut back
        cache.extend(1, 4)
        cache.shrink(1, 8, most=12)
    cache.check()
    cache.release(2)
    cache.release(1)
    cache.check()
    assert pool.n_free == pool.n_unpromised == 12


def test_another_request_without_a_promise_goes_on():
    cache = manager()
    cache.admit(1)
    cache.admit(2)
    cache.extend(1, 44)
    cache.extend(2, 4)
    with pytest.raises(OutOfPages):
        cache.extend(2, 1)
    cache.shrink(1, 8, most=8)
    cache.extend(2, 30)
    cache.check()
    cache.extend(1, 4)                                     # beyond its most it takes what is nobody's, while there is such
    with pytest.raises(OutOfPages):
        cache.extend(1, 12)
    cache.check()


def test_a_most_within_the_pages_that_stay():
    cache = manager()
    cache.admit(1, 20, 4)
    cache.extend(1, 11)
    cache.shrink(1, 9, most=10)                            # three pages either way, and two were promised beside them
    assert len(cache.table(0, 1)) == 3 and cache.groups[0].pool.n_promised == 0
    cache.check()


def test_a_bound_known_from_the_start():
    """Admitted with its budget and a step's tokens, a request of any length holds no more pages than that."""
    cache = manager()
    cache.admit(1, 12, 4)
    assert cache.groups[0].pool.n_unpromised == 9
    at = 0
    for n in [4] * 3 + [1] * 30:
        cache.extend(1, n)
        at += n
        if cache.lengths[1] > 8:
            cache.shrink(1, 8)
        assert cache.groups[0].pool.n_unpromised == 9
    assert at == 42
    cache.check()


def test_refusals():
    cache = manager()
    cache.admit(1, 20, 4)
    cache.extend(1, 11)
    with pytest.raises(ValueError):
        cache.shrink(1, 9, most=8)
    assert cache.lengths[1] == 11 and len(cache.table(0, 1)) == 3
    pool = PagePool(4)
    pool.open(7, 2)
    with pytest.raises(ValueError):
        pool.limit_promise(7, -1)
    with pytest.raises(KeyError):
        pool.limit_promise(8, 1)
    pool.limit_promise(7, 3)                               # never more than there was
    assert pool.n_promised == 2
    pool.audit()
