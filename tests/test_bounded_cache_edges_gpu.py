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


def compare(got, want, bound):
    """How many times the bound a result is off at worst."""
    return float(((got - want).abs() / bound).max())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [0.0, -0.11])
def test_scales_that_are_not_positive(hip, dtype, scale):
    """Every key alike, and the largest product the least weight: by the kernels that take any scale."""
    lens, starts, dim = [33, 600, 300], [32, 599, 260], 64
    ctx, cache = Ctx([1, 1, 40], lens), Cache(lens, 2, 16, dim, dtype)
    qkv = rnd(ctx.n_tokens, 4 * dim, dtype=dtype, seed=8)
    before = cache.weights.double()
    out = hip.weighed_attention(qkv, 4, 2, dim, scale, ctx, cache).double().view(-1, 4, dim)
    q, cu, half = qkv.double().view(-1, 4, dim), ctx.cu_q.tolist(), torch.finfo(dtype).eps / 2
    for s, length in enumerate(lens):
        k, v = cache.rows(s, length)
        for g in range(2):
            grown, size, rows = torch.zeros(length, dtype=torch.float64, device=DEV), 0.0, slice(cu[s], cu[s + 1])
            for h in (2 * g, 2 * g + 1):
                o, p, _ = attended(q[rows, h], k[g], v[g], starts[s], scale, None)
                terms = float((q[rows, h].abs() @ k[g].abs().T).max() * abs(scale))
                rel = 2 * (dim + 8) * terms * STEP32 + (length + 80) * STEP32 + 8 * STEP32 * (terms + 8)      # as in check_weighed
                assert compare(out[rows, h], o, half * o.abs() + (p @ v[g].abs()) * (2 * rel + 1.01 * half) + 1e-30) <= 1
                grown, size = grown + p.sum(0), max(size, rel)
            want = grown + torch.where(torch.arange(length, device=DEV) < starts[s], before[s, g, :length], 0.0)
            count = 2 * ctx.q_lens[s]
            assert compare(cache.weights[s, g, :length].double(), want, grown * (2 * size + count * STEP32) + want * 4 * STEP32 + 1e-30) <= 1


@pytest.mark.parametrize("q_lens,kv_lens,heads,kv,dim", [([1] * 3, [33, 1, 700], 8, 2, 128), ([1, 60, 3], [40, 60, 500], 6, 2, 64), ([1, 20], [90, 200], 4, 1, 256)])
def test_bfloat16_without_its_matrix_cores(hip, q_lens, kv_lens, heads, kv, dim):
    ctx, cache = Ctx(q_lens, kv_lens), Cache(kv_lens, kv, 16, dim, torch.bfloat16)
    qkv = rnd(ctx.n_tokens, heads * dim, dtype=torch.bfloat16, seed=8)
    hip.use_mfma_attention = False
    try:
        check_weighed(hip, ctx, cache, qkv, heads, dim ** -0.5)
    finally:
        hip.use_mfma_attention = True


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_requests_sums_from_its_first_token_on(hip, dtype):
    """A prompt, tokens and a portion with evictions between, each operator against its definition on what the one before it left, and the sums
    against a list per head that is kept in 64 bits and never takes a number from the kernels.  The bounds are relative to every single sum, so that
    sums of another head, of too few heads or of none are beyond them: the list's own mistakes show it."""
    heads, kv, dim, budget, first, last, scale = 6, 2, 64, 96, 2, 24, 0.125
    group, sections, pages = heads // kv, (12, 10, 10), 16
    cache = Cache([256], kv, pages, dim, dtype)
    cache.weights.fill_(math.nan)
    cos, sin = angles(400, 32)
    held = [torch.zeros(2, 0, dtype=torch.float64, device=DEV) for _ in range(kv)]      # per head: sums, and how far the kernels' may be off
    length = at = 0
    for n in [150] + [1] * 10 + [30] + [1] * 5:
        token = torch.arange(at, at + n, dtype=torch.int32)
        where = torch.stack([token, token // 2, token % 7]).to(DEV)
        at, length = at + n, length + n
        ctx = Ctx([n], [length])
        qkv = rnd(n, (heads + 2 * kv) * dim, dtype=dtype, seed=at)
        turned, off = rotated(qkv, heads + kv, dim, sections, cos, sin, where, "blocks", "half")
        off = off + (torch.finfo(dtype).eps / 2 * (turned.abs() + off) if dtype != torch.float32 else 0)
        values = qkv[:, (heads + kv) * dim:].double().view(n, kv, dim)
        hip.rope_axes_kv_write(qkv, heads, kv, dim, sections, cos, sin, where, ctx, cache)
        q = qkv[:, :heads * dim].double().view(n, heads, dim)
        k, v = cache.rows(0, length)
        assert ((q - turned[:, :heads]).abs() <= off[:, :heads]).all()
        assert ((k[:, length - n:].transpose(0, 1) - turned[:, heads:]).abs() <= off[:, heads:]).all()
        assert torch.equal(v[:, length - n:].transpose(0, 1), values)
        check_weighed(hip, ctx, cache, qkv, heads, scale)
        got = cache.weights[0, :, :length].double()
        for g in range(kv):
            grown, rel = [], 0.0
            for h in range(g * group, (g + 1) * group):
                _, p, terms = attended(q[:, h], k[g], v[g], length - n, scale, None)
                grown.append(p.sum(0))
                rel = max(rel, float(2 * (dim + 8) * terms * STEP32 + (length + 80) * STEP32 + 8 * STEP32 * (terms + 8)))      # as in check_weighed
            held[g] = torch.cat([held[g], torch.zeros(2, n, dtype=torch.float64, device=DEV)], 1)
            short = held[g][0] + sum(grown[1:])
            held[g][0] += sum(grown)
            held[g][1] += sum(grown) * (2 * rel + n * group * STEP32) + held[g][0] * 4 * STEP32
            sums, bound = held[g][0], held[g][1] + 1e-30
            assert compare(got[g], sums, bound) <= 1
            for wrong in (short, sums.roll(1), torch.zeros_like(sums), got[1 - g]):
                assert compare(got[g], wrong, bound) > 1
        if length > budget:
            own = cache.weights[0, :, :length].tolist()
            kept, lengths = check_evict(hip, ctx, cache, budget, first, last)
            for g in range(kv):
                lay = layout(own[g], length, budget, first, last)
                assert kept[0, g].tolist() == lay
                # what went has no more weight, by the list, than what stayed
                gone = sorted(set(range(length)) - set(lay))
                between = [j for j in lay if first <= j < length - last]
                assert float((held[g][0] - held[g][1])[gone].max()) <= float((held[g][0] + held[g][1])[between].min())
                held[g] = held[g][:, lay]
            length = int(lengths[0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_decoding_in_the_cache_managers_pages_has_the_bits_that_it_has_alone(hip, dtype):
    """Requests that decode side by side, their caches cut to a budget and pages that one gives back taken by another: from their prompts (taken
    one by one) on, every result, choice and sum has the bits that the request gets alone."""
    from simple_inference_amd.cache import CacheManager
    from simple_inference_amd.parts.model import CacheLayout
    from simple_inference_amd.parts.plan import PagedKVNeed
    heads, kv, dim, page, budget = 4, 2, 64, 16, 64
    cos, sin = angles(500, 32)
    prompts = {0: 100, 1: 30, 2: 63}

    def serve(requests):
        plan = CacheLayout([PagedKVNeed(kv, dim, None)], [1], [(0, 0)], [], [None])
        books = CacheManager(plan, page_size=page, num_pages=24, max_running=3, dtype=dtype, device=DEV)
        weights = torch.full((4, kv, 256), math.nan, device=DEV)
        seen, outs = {r: 0 for r in requests}, {r: [] for r in requests}

        def step(entries):
            q_lens, lens = [n for _, n in entries], [books.extend(r, n) + n for r, n in entries]
            ctx = Ctx(q_lens, lens, [books.slot(r) for r, _ in entries])
            tables = [books.table(0, r) for r, _ in entries]
            width = max(map(len, tables))
            layer = books.layer_caches([torch.tensor([t + [-1] * (width - len(t)) for t in tables], dtype=torch.int32, device=DEV)])[0]
            layer.weights = weights
            rows = [rnd(n, (heads + 2 * kv) * dim, dtype=dtype, seed=1000 * r + seen[r]) for r, n in entries]
            where = torch.cat([torch.arange(seen[r], seen[r] + n, dtype=torch.int32) for r, n in entries])
            qkv, where = torch.cat(rows), torch.stack([where, where // 2, where // 3]).to(DEV)
            hip.rope_axes_kv_write(qkv, heads, kv, dim, (12, 10, 10), cos, sin, where, ctx, layer)
            out = hip.weighed_attention(qkv, heads, kv, dim, 0.125, ctx, layer)
            kept, _ = hip.evict_cache(ctx, layer, budget, keep_first=2, keep_last=16)
            for s, (r, n) in enumerate(entries):
                outs[r].append((out[ctx.cu_q[s]:ctx.cu_q[s + 1]].clone(), kept[s].clone(), weights[books.slot(r), :, :min(lens[s], budget)].clone()))
                seen[r] += n
                if lens[s] > budget:
                    books.shrink(r, budget)
            books.check()

        for r in requests:
            books.admit(r)
            step([(r, prompts[r])])
        for _ in range(8):
            step([(r, 1) for r in requests])
        return outs

    together = serve([0, 1, 2])
    for r in prompts:
        for got, want in zip(together[r], serve([r])[r]):
            assert all(torch.equal(a, b) for a, b in zip(got, want))
