"""Where the operators of a bounded cache meet what a step may also hold: sequences without places, rows that are no numbers, short
sequences beside a long one, and a request's sums followed from its first token to its last."""

import math

import pytest
import torch

from test_bounded_cache_gpu import DEV, DTYPES, STEP32, Cache, Ctx, angles, attended, check_evict, check_weighed, layout, rnd, rotated

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    from simple_inference_amd.kernels import HipKernels
    return HipKernels()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sinks", [None, 1.5, -math.inf])
@pytest.mark.parametrize("dim,vdim,page", [(64, 64, 16), (20, 20, 12), (36, 36, 4), (200, 200, 16), (64, 48, 16)])
def test_sequences_without_places(hip, dtype, sinks, dim, vdim, page):
    """Their rows are zeros and nothing of theirs changes, whichever kernel takes them; the others are what they are without them."""
    ctx, cache = Ctx([1] * 4, [0, 3, 0, 70], [2, 0, 5, 1]), Cache([0, 3, 0, 70], 2, page, dim, dtype, value_dim=vdim, n_slots=6)
    qkv = rnd(4, 4 * dim, dtype=dtype, seed=3)
    sinks = None if sinks is None else torch.tensor([sinks, 0.0, sinks, 0.5], device=DEV)
    before = cache.weights.clone()
    out = check_weighed(hip, ctx, cache, qkv, 4, dim ** -0.5, sinks=sinks, poison=False)
    assert torch.equal(out[[0, 2]], torch.zeros_like(out[[0, 2]]))
    assert torch.equal(cache.weights[[2, 5, 3, 4]], before[[2, 5, 3, 4]])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q,length,heads,kv,dim,page", [(50, 50, 4, 2, 64, 16), (300, 420, 6, 2, 128, 16), (90, 400, 2, 1, 256, 32), (65, 65, 4, 2, 22, 12),
                                                        (600, 601, 8, 1, 80, 8)])
def test_a_row_that_is_no_number_spoils_only_what_it_sees(hip, dtype, q, length, heads, kv, dim, page):
    """One token's query of the first head is NaN: the sums of the first group's keys up to that token's place are, those beyond are not."""
    ctx, cache = Ctx([q], [length]), Cache([length], kv, page, dim, dtype)
    qkv, at, start = rnd(q, heads * dim, dtype=dtype, seed=8), q // 3, length - q
    other, before = qkv.clone(), cache.weights.clone()
    qkv[at, :dim] = math.nan
    other[at, :dim] = 0
    scale = dim ** -0.5
    out = hip.weighed_attention(qkv, heads, kv, dim, scale, ctx, cache)
    got = cache.weights.clone()
    assert out[at, :dim].isnan().all()
    assert got[0, 0, :start + at + 1].isnan().all()
    cache.weights.copy_(before)
    want = check_weighed(hip, ctx, cache, other, heads, scale, poison=False)      # a query of zeros weighs no key beyond its place either
    out[at, :dim] = want[at, :dim]
    assert torch.equal(out, want)
    assert torch.equal(got[0, 0, start + at + 1:], cache.weights[0, 0, start + at + 1:]) and torch.equal(got[0, 1:], cache.weights[0, 1:])


def grown_by(call):
    """Bytes of GPU memory that a call has at most beside what there was before it."""
    call()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    there = torch.cuda.memory_allocated()
    call()
    return torch.cuda.max_memory_allocated() - there


@pytest.mark.parametrize("dtype", DTYPES)
def test_short_rows_beside_a_long_run(hip, dtype):
    """Single tokens over some tens of keys, one of them over nothing but itself, beside a portion over thousands: right, and with workspaces for
    the keys and rows that there are."""
    q_lens, lens, heads, kv, dim = [1] * 40 + [300], [1 + 7 * i % 60 for i in range(40)] + [5000], 8, 2, 64
    ctx, cache = Ctx(q_lens, lens), Cache(lens, kv, 16, dim, dtype)
    ctx.max_single_kv_len = max(lens[:40])
    qkv = rnd(ctx.n_tokens, heads * dim, dtype=dtype, seed=8)
    check_weighed(hip, ctx, cache, qkv, heads, 0.125)
    # results, statistics, scores of 40 rows over at most 64 keys with their states, and pieces of the run's rows over its keys: some 4 (8 in
    # float32) of 64 query rows for each of 5,000 keys and 2 heads
    rows = qkv.numel() * qkv.element_size() + ctx.n_tokens * heads * 4 + 40 * heads * (64 + 66) * 4
    assert grown_by(lambda: hip.weighed_attention(qkv, heads, kv, dim, 0.125, ctx, cache)) < 2 * rows + 20 * 5200 * kv * 4
    out = hip.weighed_attention(qkv, heads, kv, dim, 0.125, ctx, cache)
    ctx.max_single_kv_len = 0                    # not known: the step's own bound
    assert torch.equal(hip.weighed_attention(qkv, heads, kv, dim, 0.125, ctx, cache), out)


def test_a_group_of_more_heads_than_a_chunk_has_rows(hip):
    """Float heads, 65 and 70 of them a key/value head: single tokens have chunks too."""
    for heads, kv in ((65, 1), (140, 2)):
        ctx, cache = Ctx([1, 1, 20], [300, 7, 90]), Cache([300, 7, 90], kv, 16, 32, torch.float32)
        check_weighed(hip, ctx, cache, rnd(ctx.n_tokens, heads * 32, seed=8), heads, 32 ** -0.5)


def test_many_short_rows_in_float32(hip):
    """More pieces of work than a row of the grid has: 5,000 single tokens, and a run, under a bound of 2,000 keys."""
    q_lens, lens = [1] * 5000 + [50], [1 + i % 37 for i in range(5000)] + [2000]
    ctx, cache = Ctx(q_lens, lens), Cache(lens, 1, 16, 16, torch.float32)
    qkv = rnd(ctx.n_tokens, 16, seed=8)
    before = cache.weights.clone()
    out = hip.weighed_attention(qkv, 1, 1, 16, 0.25, ctx, cache)
    got = cache.weights.clone()
    for s in (0, 1, 36, 37, 2500, 4094, 4095, 4096, 4999, 5000):      # alone they have the same bits, or a run's sums up to their order
        alone = Cache([lens[s]], 1, 16, 16, torch.float32)
        alone.k_pages, alone.v_pages, alone.block_table = cache.k_pages, cache.v_pages, cache.block_table[s:s + 1].contiguous()
        alone.weights = before[s:s + 1].clone()
        rows = slice(int(ctx.cu_q[s]), int(ctx.cu_q[s + 1]))
        one = check_weighed(hip, Ctx([q_lens[s]], [lens[s]], [0]), alone, qkv[rows].contiguous(), 1, 0.25, poison=False)
        assert torch.equal(one, out[rows])
        if q_lens[s] == 1:
            assert torch.equal(alone.weights[0], got[s])
        else:
            torch.testing.assert_close(alone.weights[0], got[s], rtol=50 * 2 * STEP32, atol=0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_request_with_an_adopted_prefix(hip, dtype):
    """Its sums hold what its own tokens gave the adopted places, and nothing of whoever had its slot before; once it is the pages' only holder,
    eviction goes by them."""
    from simple_inference_amd.cache import CacheManager
    from simple_inference_amd.parts.model import CacheLayout
    from simple_inference_amd.parts.plan import PagedKVNeed
    heads, kv, dim, page = 4, 2, 64, 16
    plan = CacheLayout([PagedKVNeed(kv, dim, None)], [1], [(0, 0)], [], [None])
    books = CacheManager(plan, page_size=page, num_pages=24, max_running=3, dtype=dtype, device=DEV)
    books.keep_weights(160)
    cos, sin = angles(200, 32)

    def layer_of(req):
        return books.layer_caches([torch.tensor([books.table(0, req)], dtype=torch.int32, device=DEV)])[0]

    def step(req, n):
        length = books.extend(req, n) + n
        ctx, layer = Ctx([n], [length], [books.slot(req)]), layer_of(req)
        qkv = rnd(n, (heads + 2 * kv) * dim, dtype=dtype, seed=100 * req + length)
        hip.rope_axes_kv_write(qkv, heads, kv, dim, (32,), cos, sin, ctx.positions[None].contiguous(), ctx, layer)
        view = Cache([length], kv, page, dim, dtype)      # for its way of looking at pages
        view.k_pages, view.v_pages, view.block_table, view.weights = layer.k_pages, layer.v_pages, layer.block_table, layer.weights
        check_weighed(hip, ctx, view, qkv, heads, 0.125, poison=False)
        return ctx, view

    books.admit(1)
    step(1, 70)
    books.groups[0].weights[:, 1:] = math.nan             # what others left in the other rows
    slot = books.admit(2, shared_pages=books.table(0, 1)[:4])
    ctx, view = step(2, 30)
    got = view.weights[slot, :, :94].double()
    assert torch.allclose(got.sum(-1), torch.full((kv,), 30.0 * heads / kv, dtype=torch.float64, device=DEV), rtol=1e-4)
    books.release(1)
    assert books.owns_pages(2)
    check_evict(hip, ctx, view, 40, 2, 8)
    books.shrink(2, 40)
    books.check()
