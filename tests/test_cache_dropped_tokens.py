"""A request whose cache has dropped tokens: what its places no longer stand for (no GPU)."""

import pytest

from helpers import TINIES, make_runner, random_tokens, write_tiny_model
from simple_inference_amd.cache import PrefixCache
from simple_inference_amd.engine import StepEntry
from test_cache_shrink import manager


def test_pages_of_a_request_that_dropped_tokens_are_no_prefix():
    cache = manager(num_pages=24)
    prefixes = PrefixCache(cache, max_pages=24)
    tokens = list(range(40))
    cache.admit(1)
    cache.extend(1, 12)
    prefixes.insert_pages_of(1, tokens[:12])
    assert prefixes.match(tokens) == cache.table(0, 1)[:3]
    # another request with the same prompt, which has pages of its own (it was admitted before the first had written its)
    cache.admit(2)
    cache.extend(2, 24)
    prefixes.insert_pages_of(2, tokens[:12])                  # known already: nothing of it is pinned
    assert cache.owns_pages(2) and not cache.has_shrunk(2)
    cache.shrink(2, 10)
    assert cache.has_shrunk(2) and not cache.has_shrunk(1)
    cache.extend(2, 16)                                       # its tokens 24 .. 39, in places 10 .. 25
    prefixes.insert_pages_of(2, tokens)
    assert prefixes.match(tokens + [0]) == cache.table(0, 1)[:3] and cache.owns_pages(2)
    cache.check()
    cache.release(2)
    cache.admit(2)                                            # the id again, of a request that dropped nothing
    assert not cache.has_shrunk(2)
    cache.extend(2, 24)
    prefixes.insert_pages_of(2, tokens[:24])
    assert prefixes.match(tokens) == cache.table(0, 1)[:3] + cache.table(0, 2)[3:6]
    cache.reset()
    assert not cache.has_shrunk(2)


def test_a_request_that_is_cut_back_to_what_it_has_dropped_nothing():
    cache = manager()
    cache.admit(1)
    cache.extend(1, 9)
    cache.shrink(1, 9)
    assert not cache.has_shrunk(1)
    cache.shrink(1, 8)
    cache.shrink(1, 8)
    assert cache.has_shrunk(1)


def test_a_step_does_not_rotate_by_places(tmp_path):
    """Tokens of such a request are taken only with positions of their own; nothing is booked for those that are refused."""
    folder = write_tiny_model(tmp_path, TINIES["b"], seed=3)
    runner, cache, cfg = make_runner(folder, "twins", 8, 64)
    tokens = random_tokens(cfg.vocab_size, 40, seed=1)
    for req in (0, 1):
        cache.admit(req)
        runner.run([StepEntry(req, tokens[:30], [29])])
    cache.shrink(0, 12)
    for entries in ([StepEntry(0, tokens[30:31])], [StepEntry(1, tokens[30:32]), StepEntry(0, tokens[30:33], [2])]):
        with pytest.raises(ValueError, match="dropped tokens"):
            runner.run(entries)
    assert (cache.lengths[0], cache.lengths[1]) == (12, 30)
    runner.run([StepEntry(1, tokens[30:31], [0])])
    ctx = runner.build_context([StepEntry(0, tokens[30:32], extra={"time": [30, 31]}), StepEntry(1, tokens[31:32], extra={"time": [31]})])
    assert ctx.positions.tolist() == [31, 12, 13] and ctx.extra["time"].tolist() == [31, 30, 31]
    cache.check()
