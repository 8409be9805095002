"""Rotation by several axes, attention that weighs the cache and eviction by weight, each against its definition in 64 bits, and
the three together as a program uses them.

Tolerances are worst cases of the arithmetic, written where they are used: a rounding to a type is off by at most half a step,
``finfo(type).eps / 2`` of the value."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
DTYPES = [torch.float32, torch.bfloat16]
STEP32 = torch.finfo(torch.float32).eps / 2


@pytest.fixture(scope="module")
def hip():
    from simple_inference_amd.kernels import HipKernels
    return HipKernels()


def rnd(*shape, dtype=torch.float32, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


class Ctx:
    """The fields of a step context that the kernels read."""

    def __init__(self, q_lens, kv_lens, slots=None, kv_bound=0):
        pos, sot, cu = [], [], [0]
        for s, (q, kv) in enumerate(zip(q_lens, kv_lens)):
            pos += list(range(kv - q, kv))      # (a sequence without places: place -1)
            sot += [s] * q
            cu.append(cu[-1] + q)
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
        self.positions, self.seq_of_token, self.cu_q, self.kv_len = i32(pos), i32(sot), i32(cu), i32(list(kv_lens))
        self.state_slots = i32(list(slots if slots is not None else range(len(q_lens))))
        self.n_tokens, self.n_seqs = len(pos), len(q_lens)
        self.max_q_len, self.max_kv_len, self.kv_bound = max(q_lens), max(kv_lens), kv_bound
        self.q_lens = list(q_lens)
        self.n_decode_seqs = next((i for i, q in enumerate(q_lens) if q != 1), len(q_lens))
        self.max_run_kv_len = max([k for q, k in zip(q_lens, kv_lens) if q > 1], default=0)


class Cache:
    """Pages in no particular order, one more than are used, with something in all of them; weights of n_slots rows."""

    def __init__(self, kv_lens, n_kv, page_size, head_dim, dtype, value_dim=None, n_slots=None, places=None, seed=0, room=0):
        self.page_size = page_size
        per = [-(-(kv + room) // page_size) for kv in kv_lens]
        n_pages = sum(per) + 1
        g = torch.Generator().manual_seed(seed)
        perm = torch.randperm(n_pages, generator=g).tolist()
        table = torch.full((len(kv_lens), max(per)), -1, dtype=torch.int32)
        for s, n in enumerate(per):
            for i in range(n):
                table[s, i] = perm.pop()
        self.spare = perm.pop()
        self.block_table = table.to(DEV)
        self.k_pages = rnd(n_pages, n_kv, page_size, head_dim, dtype=dtype, seed=seed + 1)
        self.v_pages = rnd(n_pages, n_kv, value_dim or head_dim, page_size, dtype=dtype, seed=seed + 2)
        self.weights = rnd(n_slots or len(kv_lens), n_kv, places or max(per) * page_size, seed=seed + 3).abs()

    def rows(self, s, length):
        """Keys and values of a sequence's first places in 64 bits: [n_kv, length, dim]."""
        pages = self.block_table[s, :-(-length // self.page_size)].long()
        n_kv = self.k_pages.shape[1]
        k = self.k_pages[pages].transpose(0, 1).reshape(n_kv, -1, self.k_pages.shape[3])[:, :length]
        v = self.v_pages[pages].permute(1, 0, 3, 2).reshape(n_kv, -1, self.v_pages.shape[2])[:, :length]
        return k.double(), v.double()


# -- rotation by several axes ------------------------------------------------------------------------------------

def axis_of_pair(sections, order):
    if order == "blocks":
        return [a for a, c in enumerate(sections) for _ in range(c)]
    n, left, out = len(sections), list(sections), []
    for j in range(sum(sections)):
        a = j % n
        if a and left[a]:
            left[a] -= 1
            out.append(a)
        else:
            out.append(0)
    return out


def rotated(qkv, heads, head_dim, sections, cos, sin, where, order, pairing):
    """(64-bit result, bound of its 32-bit arithmetic) of the first ``heads`` heads of the rows."""
    half = sum(sections)
    x = qkv[:, :heads * head_dim].double().view(len(qkv), heads, head_dim)
    out, off = x.clone(), torch.zeros_like(x)
    for j, a in enumerate(axis_of_pair(sections, order)):
        at = where[a].long().clamp(0, len(cos) - 1)
        c, s = cos[at, j].double()[:, None], sin[at, j].double()[:, None]
        i, k = (j, j + half) if pairing == "half" else (2 * j, 2 * j + 1)
        out[:, :, i], out[:, :, k] = x[:, :, i] * c - x[:, :, k] * s, x[:, :, k] * c + x[:, :, i] * s
        # one product rounded, then a fused multiply-add
        off[:, :, i], off[:, :, k] = STEP32 * ((x[:, :, k] * s).abs() * 2 + out[:, :, i].abs()), STEP32 * ((x[:, :, i] * s).abs() * 2 + out[:, :, k].abs())
    return out, off


def angles(rows, half):
    a = torch.outer(torch.arange(rows, dtype=torch.float64), 10000.0 ** (-torch.arange(half, dtype=torch.float64) / half))
    return a.cos().float().to(DEV), a.sin().float().to(DEV)


ROTATIONS = [
    # q lens, kv lens, heads, kv, dim, sections, order, pairing, page size
    ([1], [1], 4, 2, 64, (8, 12, 12), "blocks", "half", 16),
    ([1] * 9, [1, 2, 15, 16, 17, 31, 32, 33, 700], 6, 2, 128, (16, 24, 24), "blocks", "half", 16),
    ([37], [37], 3, 3, 64, (11, 11, 10), "cycled", "half", 16),
    ([75], [80], 8, 1, 128, (22, 21, 21), "cycled", "interleaved", 64),
    ([1, 1, 40, 17, 2], [5, 40, 49, 17, 16], 4, 2, 32, (4, 4, 4, 4), "blocks", "interleaved", 8),
    ([50, 33], [60, 33], 5, 5, 80, (20,), "blocks", "half", 16),                 # a part of the head, one axis
    ([19, 3], [19, 20], 2, 1, 36, (3, 2, 2), "cycled", "half", 12),              # nothing in eights, pages of no power of two
    ([21], [21], 2, 2, 6, (1, 1), "blocks", "interleaved", 4),
    ([130], [130], 2, 2, 256, (64, 0, 64), "blocks", "half", 32),                # an axis without pairs
    ([200, 1, 65], [264, 9, 65], 24, 8, 96, (16, 16, 16), "cycled", "half", 16),
    ([40], [43], 1, 1, 392, (98, 98), "cycled", "interleaved", 16),              # pieces that fill no wave
    ([1] * 70, [17 + i for i in range(70)], 4, 4, 192, (40, 20, 20), "blocks", "half", 8),
    ([2100], [2137], 4, 1, 64, (12, 10, 10), "blocks", "half", 16),              # long enough for workgroups of several tokens
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q_lens,kv_lens,heads,kv,dim,sections,order,pairing,page", ROTATIONS)
def test_rope_axes_kv_write(hip, dtype, q_lens, kv_lens, heads, kv, dim, sections, order, pairing, page):
    ctx, cache = Ctx(q_lens, kv_lens), Cache(kv_lens, kv, page, dim, dtype)
    n, half = ctx.n_tokens, sum(sections)
    cos, sin = angles(300, half)
    where = torch.randint(0, 300, (len(sections), n), generator=torch.Generator().manual_seed(5), dtype=torch.int32).to(DEV)
    qkv = rnd(n, (heads + 2 * kv) * dim, dtype=dtype, seed=6)
    given, keys, values = qkv.clone(), cache.k_pages.clone(), cache.v_pages.clone()
    want, off = rotated(given, heads + kv, dim, sections, cos, sin, where, order, pairing)
    bound = off + (torch.finfo(dtype).eps / 2 * (want.abs() + off) if dtype != torch.float32 else 0)
    hip.rope_axes_kv_write(qkv, heads, kv, dim, sections, cos, sin, where, ctx, cache, order=order, pairing=pairing)
    got = qkv[:, :heads * dim].double().view(n, heads, dim)
    assert ((got - want[:, :heads]).abs() <= bound[:, :heads]).all()
    assert torch.equal(qkv[:, heads * dim:], given[:, heads * dim:])       # what the rows hold of k and v stays
    # every written place, and nothing beside them
    page_of = ctx.positions.long() // page
    pages, at = cache.block_table[ctx.seq_of_token.long(), page_of].long(), ctx.positions.long() % page
    got_k = cache.k_pages[pages, :, at].double()
    assert ((got_k - want[:, heads:]).abs() <= bound[:, heads:]).all()
    values[pages, :, :, at] = given[:, (heads + kv) * dim:].view(n, kv, dim)
    assert torch.equal(cache.v_pages, values)
    keys[pages, :, at] = cache.k_pages[pages, :, at]
    assert torch.equal(cache.k_pages, keys)


def test_one_axis_at_the_places_is_the_plain_rotation(hip):
    for dtype in DTYPES:
        ctx, cache = Ctx([1, 40], [70, 45]), Cache([70, 45], 2, 16, 64, dtype)
        other = Cache([70, 45], 2, 16, 64, dtype)
        cos, sin = angles(80, 32)
        qkv = rnd(41, 8 * 64, dtype=dtype, seed=1)
        plain = qkv.clone()
        hip.rope_axes_kv_write(qkv, 4, 2, 64, (32,), cos, sin, ctx.positions[None].contiguous(), ctx, cache)
        hip.rope_kv_write(plain, 4, 2, 64, 64, cos, sin, ctx, other)
        assert torch.equal(qkv, plain) and torch.equal(cache.k_pages, other.k_pages) and torch.equal(cache.v_pages, other.v_pages)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,page", [(64, 16), (36, 12)])
def test_rotation_without_pages_and_outside_the_tables(hip, dtype, dim, page):
    """No pages to write (a layer that reads another's), pages that are none, positions that no table row has."""
    ctx, cache = Ctx([20], [20]), Cache([20], 2, page, dim, dtype)
    sections = (dim // 4, dim // 4)
    cos, sin = angles(50, dim // 2)
    where = torch.randint(-9, 90, (2, 20), generator=torch.Generator().manual_seed(3), dtype=torch.int32).to(DEV)
    qkv = rnd(20, 8 * dim, dtype=dtype, seed=4)
    same = qkv.clone()
    want, off = rotated(qkv, 4, dim, sections, cos, sin, where, "blocks", "half")
    bound = off + (torch.finfo(dtype).eps / 2 * (want.abs() + off) if dtype != torch.float32 else 0)
    q_only = qkv[:, :4 * dim].contiguous()
    hip.rope_axes_kv_write(q_only, 4, 0, dim, sections, cos, sin, where, ctx, None)
    assert ((q_only.double().view(20, 4, dim) - want).abs() <= bound).all()
    keys, values = cache.k_pages.clone(), cache.v_pages.clone()
    for bad in (-1, cache.k_pages.shape[0], 1 << 30):
        cache.block_table.fill_(bad)
        qkv = same.clone()
        hip.rope_axes_kv_write(qkv, 4, 2, dim, sections, cos, sin, where, ctx, cache)
        assert torch.equal(qkv[:, :4 * dim], q_only)
        assert torch.equal(cache.k_pages, keys) and torch.equal(cache.v_pages, values)


def test_rotation_refuses(hip):
    from simple_inference_amd.kernels import KernelError
    ctx, cache = Ctx([3], [3]), Cache([3], 2, 16, 64, torch.bfloat16)
    cos, sin = angles(8, 32)
    qkv, where = rnd(3, 8 * 64, dtype=torch.bfloat16), torch.zeros(3, 3, dtype=torch.int32, device=DEV)
    good = dict(qkv=qkv, n_heads=4, n_kv_written=2, head_dim=64, sections=(12, 10, 10), cos=cos, sin=sin, rotary_positions=where, ctx=ctx, cache=cache)
    before = qkv.clone()
    for change in (dict(sections=(12, 10, 11)), dict(sections=(12, 10)), dict(sections=()), dict(sections=(8, 8, 8, 4, 4)), dict(sections=(44, -6, -6)),
                   dict(sections=(0, 16, 16), order="cycled"), dict(order="rows"), dict(pairing="other"), dict(rotary_positions=where.long()),
                   dict(rotary_positions=where[:2]), dict(rotary_positions=where.t()[:, :3].t()[:, :2]), dict(cos=cos[:, :16]), dict(cos=cos[:4]), dict(sin=sin.double()),
                   dict(qkv=qkv.half()), dict(qkv=qkv[:2]), dict(qkv=qkv[:, ::2]), dict(n_heads=5), dict(head_dim=32), dict(qkv=qkv.cpu()),
                   dict(cos=cos[:0], sin=sin[:0]), dict(ctx=Ctx([3], [40]))):
        with pytest.raises(KernelError):
            hip.rope_axes_kv_write(**{**good, **change})
    assert torch.equal(qkv, before)


# -- attention that weighs the cache -----------------------------------------------------------------------------

def attended(q, k, v, start, scale, sinks):
    """One head: (out, weights [rows, places], size of the scores' terms) in 64 bits."""
    s = q @ k.T * scale
    mask = torch.ones_like(s, dtype=torch.bool).tril(start)
    s = s.masked_fill(~mask, -math.inf)
    top = s.amax(-1, keepdim=True)
    e = (s - top).exp()
    total = e.sum(-1, keepdim=True) + (0 if sinks is None else (sinks - top).exp())
    p = e / total
    return p @ v, p, (q.abs() @ k.abs().T * scale).max()


def check_weighed(hip, ctx, cache, qkv, heads, scale, sinks=None, poison=True):
    kv, dim, vdim = cache.k_pages.shape[1], cache.k_pages.shape[3], cache.v_pages.shape[2]
    dtype, group = qkv.dtype, heads // cache.k_pages.shape[1]
    cu, lens, slots = ctx.cu_q.tolist(), ctx.kv_len.tolist(), ctx.state_slots.tolist()
    if poison:      # whatever lies where the step writes is no part of the sums
        for s, length in enumerate(lens):
            if length > 0:
                cache.weights[slots[s], :, length - (cu[s + 1] - cu[s]):length] = math.nan
    before = cache.weights.clone()
    out = hip.weighed_attention(qkv, heads, kv, dim, scale, ctx, cache, value_dim=vdim, sinks=sinks)
    assert out.shape == (ctx.n_tokens, heads * vdim) and out.dtype == dtype
    q = qkv.double()[:, :heads * dim].view(ctx.n_tokens, heads, dim)
    got_out, touched = out.double().view(ctx.n_tokens, heads, vdim), torch.zeros_like(before, dtype=torch.bool)
    for s, length in enumerate(lens):
        if length <= 0:
            continue
        k, v = cache.rows(s, length)
        rows, start = slice(cu[s], cu[s + 1]), length - (cu[s + 1] - cu[s])
        for g in range(kv):
            add, size, count = torch.zeros(length, dtype=torch.float64, device=DEV), 0.0, 0
            for h in range(g * group, (g + 1) * group):
                o, p, terms = attended(q[rows, h], k[g], v[g], start, scale, None if sinks is None else sinks[h].double())
                # a score: dim products and sums, the scale, the change of base, its place beside the row's statistic, whose own error is a
                # score's and that of a sum of `length` terms; an exponential of the hardware is off by an ulp
                rel = float(2 * (dim + 8) * terms * STEP32 + (length + 80) * STEP32 + 8 * STEP32 * (terms + 8))
                half = torch.finfo(dtype).eps / 2
                spread = p @ v[g].abs()
                bound = half * o.abs() + spread * (rel * 2 + (half if dtype != torch.float32 else 0) * 1.01) + 1e-30
                worst = ((got_out[rows, h] - o).abs() / bound).max()
                assert worst <= 1, f"sequence {s} head {h}: {float(worst)} times the bound"
                add += p.sum(0)
                size = max(size, rel)
                count += p.shape[0]
            old = before[slots[s], g, :length].double()
            old[start:] = 0
            want, got = old + add, cache.weights[slots[s], g, :length].double()
            bound = add * (2 * size + count * STEP32) + want * 4 * STEP32 + 1e-30
            worst = ((got - want).abs() / bound).max()
            assert worst <= 1, f"sequence {s} weights of head {g}: {float(worst)} times the bound"
            touched[slots[s], g, :length] = True
    same = (cache.weights == before) | (cache.weights.isnan() & before.isnan())
    assert (same | touched).all()        # rows and places of nobody in the step stay
    return out


ATTENTIONS = [
    # q lens, kv lens, heads, kv, dim, page size
    ([1], [1], 4, 2, 64, 16),
    ([1], [40], 32, 8, 64, 16),
    ([1] * 10, [1, 2, 31, 32, 33, 63, 64, 65, 127, 300], 6, 2, 128, 16),
    ([1] * 3, [511, 512, 1100], 8, 8, 64, 16),                     # a query head a key/value head
    ([1] * 2, [700, 65], 16, 1, 128, 32),                          # sixteen
    ([1] * 2, [90, 600], 40, 2, 32, 16),                           # twenty: more than a launch's columns
    ([1], [4500], 4, 1, 128, 16),                                  # many splits
    ([1] * 2, [3000, 100], 2, 2, 256, 64),
    ([1] * 2, [260, 33], 10, 2, 80, 16),
    ([1], [77], 4, 2, 16, 8),
    ([37], [37], 4, 2, 64, 16),
    ([100, 3], [100, 70], 6, 2, 128, 16),                          # a portion of few tokens over a past
    ([300], [300], 4, 1, 96, 16),
    ([520], [700], 3, 3, 128, 16),
    ([65], [400], 2, 1, 256, 16),
    ([129], [129], 20, 1, 48, 32),
    ([1, 1, 200, 33], [90, 700, 260, 33], 8, 2, 128, 16),          # decoded tokens beside portions
    ([1, 1, 300], [150, 260, 300], 32, 8, 64, 16),
    ([5, 1], [5, 9], 2, 1, 20, 12),                                # odd heads, pages of no power of two
    ([1, 30], [50, 41], 3, 3, 36, 4),
    ([70, 1, 9], [300, 5, 9], 6, 2, 22, 12),                       # heads that are not in fours
    ([1, 45], [90, 200], 4, 2, 200, 16),
    ([1] * 3, [0, 3, 0], 4, 2, 64, 16),                            # sequences without places
    ([40, 300], [17000, 301], 2, 1, 32, 64),                       # more blocks of keys than a wave has lanes
    ([1, 3], [40, 20], 260, 1, 16, 16),                            # more query heads a key/value head than the joining kernel takes
    ([2] * 70, [5 + i for i in range(70)], 2, 2, 64, 16),          # many short runs
    ([1], [130], 4, 4, 256, 16),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q_lens,kv_lens,heads,kv,dim,page", ATTENTIONS)
def test_weighed_attention(hip, dtype, q_lens, kv_lens, heads, kv, dim, page):
    slots = torch.randperm(len(q_lens) + 2, generator=torch.Generator().manual_seed(9)).tolist()[:len(q_lens)]
    ctx = Ctx(q_lens, kv_lens, slots)
    cache = Cache(kv_lens, kv, page, dim, dtype, n_slots=len(q_lens) + 2, places=max(kv_lens) + 5)
    qkv = rnd(ctx.n_tokens, (heads + 2 * kv) * dim, dtype=dtype, seed=8)
    check_weighed(hip, ctx, cache, qkv, heads, dim ** -0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q_lens,kv_lens,heads,kv,dim,vdim,page", [([1, 45], [200, 60], 6, 2, 64, 32, 16), ([1, 1], [40, 600], 4, 4, 48, 96, 8),
                                                                  ([9], [30], 2, 1, 640, 512, 16), ([1, 400], [900, 450], 8, 2, 128, 64, 16)])
def test_weighed_attention_with_values_of_another_width(hip, dtype, q_lens, kv_lens, heads, kv, dim, vdim, page):
    ctx, cache = Ctx(q_lens, kv_lens), Cache(kv_lens, kv, page, dim, dtype, value_dim=vdim)
    check_weighed(hip, ctx, cache, rnd(ctx.n_tokens, heads * dim, dtype=dtype, seed=8), heads, dim ** -0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1], [40, 1300]), ([1, 150], [600, 200])])
def test_weighed_attention_with_sinks(hip, dtype, q_lens, kv_lens):
    """A sink takes weight that no place gets; queries that agree with one key nearly whole, and queries of zeros (every key alike)."""
    ctx, cache = Ctx(q_lens, kv_lens), Cache(kv_lens, 2, 16, 64, dtype)
    qkv = rnd(ctx.n_tokens, 8 * 64, dtype=dtype, seed=8)
    qkv[0, :64] *= 8
    qkv[-1, 64:128] = 0
    sinks = torch.tensor([-3.0, 0.5, 6.0, 20.0], device=DEV)
    check_weighed(hip, ctx, cache, qkv, 4, 0.125, sinks=sinks)


@pytest.mark.parametrize("dtype", DTYPES)
def test_weights_grow_over_steps(hip, dtype):
    """Every row's weights sum to one: after a prompt and some tokens the sums of a head's group sum to queries times heads."""
    heads, kv, dim = 6, 2, 64
    cache = Cache([90], kv, 16, dim, dtype)
    cache.weights.fill_(math.nan)
    total = 0
    for q, length in ((40, 40), (1, 41), (1, 42), (30, 72), (1, 73)):
        ctx = Ctx([q], [length])
        check_weighed(hip, ctx, cache, rnd(q, heads * dim, dtype=dtype, seed=length), heads, dim ** -0.5, poison=False)
        total += q * heads // kv
        assert torch.allclose(cache.weights[0, :, :length].double().sum(-1), torch.tensor(float(total), dtype=torch.float64, device=DEV), rtol=1e-4)


@pytest.mark.parametrize("dtype", DTYPES)
def test_weighed_attention_of_a_sequence_does_not_depend_on_its_batch(hip, dtype):
    """Decoded tokens: the same bits alone and among others, under whatever bound of the lengths."""
    lens, heads, kv, dim = [33, 900, 1, 2300, 64], 8, 2, 128
    cache = Cache(lens, kv, 16, dim, dtype)
    q = rnd(len(lens), heads * dim, dtype=dtype, seed=4)
    kept = cache.weights.clone()
    out = hip.weighed_attention(q, heads, kv, dim, 0.1, Ctx([1] * len(lens), lens), cache)
    together = cache.weights.clone()
    for s, length in enumerate(lens):
        cache.weights.copy_(kept)
        alone = Cache([1], kv, 16, dim, dtype)
        alone.k_pages, alone.v_pages, alone.block_table, alone.weights = cache.k_pages, cache.v_pages, cache.block_table[s:s + 1].contiguous(), cache.weights
        one = hip.weighed_attention(q[s:s + 1].contiguous(), heads, kv, dim, 0.1, Ctx([1], [length], [s], kv_bound=2304), alone)
        assert torch.equal(one[0], out[s]) and torch.equal(cache.weights[s, :, :length], together[s, :, :length])


@pytest.mark.parametrize("dtype", DTYPES)
def test_weighed_attention_beside_what_it_must_not_read(hip, dtype):
    """Rows of q inside a wider matrix; numbers without bounds in keys behind a sequence's places, in weights of others; a row that is no slot's."""
    lens, heads, kv, dim = [50, 700], 4, 2, 64
    ctx, cache = Ctx([1, 1], lens, [0, 3]), Cache(lens, kv, 16, dim, dtype, n_slots=5)
    qkv = rnd(2, (heads + 2 * kv + 4) * dim, dtype=dtype, seed=4)
    cache.weights[1] = math.inf
    cache.weights[4] = math.nan
    for s, length in enumerate(lens):
        page = int(cache.block_table[s, length // 16])
        cache.k_pages[page, :, length % 16:] = math.inf
    check_weighed(hip, ctx, cache, qkv, heads, 0.125)
    before = cache.weights.clone()
    ctx.state_slots[0], ctx.state_slots[1] = -1, 5
    hip.weighed_attention(qkv, heads, kv, dim, 0.125, ctx, cache)
    assert torch.equal(torch.nan_to_num(cache.weights, 7.0), torch.nan_to_num(before, 7.0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q_lens,kv_lens,heads,kv,dim,page", [
    ([1, 45], [33, 45], 4, 2, 64, 16), ([1, 1, 300], [31, 700, 1001], 6, 2, 128, 32), ([2100], [2100], 2, 1, 128, 64), ([700, 3, 30], [700, 2603, 61], 8, 2, 80, 8),
    ([17, 65], [17, 333], 4, 1, 256, 16), ([9, 520], [9, 521], 2, 2, 16, 128), ([40, 33], [75, 33], 4, 2, 100, 16), ([1, 6], [7, 9], 2, 2, 48, 4)])
def test_weighed_attention_whatever_lies_behind_the_places(hip, dtype, q_lens, kv_lens, heads, kv, dim, page):
    """Keys and values behind every sequence's places, and pages that are nobody's, without bounds or no numbers."""
    ctx, cache = Ctx(q_lens, kv_lens), Cache(kv_lens, kv, page, dim, dtype, room=page)
    spare = torch.ones(cache.k_pages.shape[0], page, dtype=torch.bool, device=DEV)
    for s, length in enumerate(kv_lens):
        at = torch.arange(length, device=DEV)
        spare[cache.block_table[s].long()[at // page], at % page] = False
    odd = torch.where(rnd(*spare.shape, seed=6) < 0, math.nan, math.inf).to(dtype)
    cache.k_pages.copy_(torch.where(spare[:, None, :, None], odd[:, None, :, None], cache.k_pages))
    cache.v_pages.copy_(torch.where(spare[:, None, None, :], odd[:, None, None, :], cache.v_pages))
    check_weighed(hip, ctx, cache, rnd(ctx.n_tokens, heads * dim, dtype=dtype, seed=8), heads, dim ** -0.5)


def test_weighed_attention_refuses(hip):
    from simple_inference_amd.kernels import KernelError
    ctx, cache = Ctx([1, 4], [40, 20]), Cache([40, 20], 2, 16, 64, torch.bfloat16)
    qkv = rnd(5, 8 * 64, dtype=torch.bfloat16)
    good = dict(qkv=qkv, n_heads=4, n_kv_heads=2, head_dim=64, scale=0.125, ctx=ctx, cache=cache)
    weights = cache.weights.clone()
    for change in (dict(n_heads=3), dict(n_kv_heads=0), dict(head_dim=0), dict(head_dim=32), dict(qkv=qkv[:4]), dict(qkv=qkv[:, :128]), dict(qkv=qkv.half()),
                   dict(qkv=qkv.float()), dict(value_dim=32), dict(sinks=torch.zeros(3, device=DEV)), dict(sinks=torch.zeros(4, device=DEV).half()), dict(qkv=qkv.cpu())):
        with pytest.raises(KernelError):
            hip.weighed_attention(**{**good, **change})
    for bad in (None, weights[:, :1].contiguous(), weights[:, :, :39].contiguous(), weights.double(), weights.transpose(0, 1), weights[0]):
        cache.weights = bad
        with pytest.raises(KernelError):
            hip.weighed_attention(**good)
        with pytest.raises(KernelError):
            hip.evict_cache(ctx, cache, 8)
    cache.weights = weights
    ctx.state_slots = ctx.state_slots[:1]
    with pytest.raises(KernelError):
        hip.weighed_attention(**good)


# -- eviction ------------------------------------------------------------------------------------------------------

def layout(w, length, budget, first, last):
    """The old places, in the order in which they lie afterwards."""
    if length <= budget:
        return list(range(length))
    value = lambda j: -math.inf if math.isnan(w[j]) else w[j]
    between = sorted(range(first, length - last), key=lambda j: (-value(j), j))[:budget - first - last]
    body, edge = sorted(list(range(first)) + between), budget - last
    fill = iter([j for j in body if j >= edge])
    stay = {j for j in body if j < edge}
    return [j if j in stay else next(fill) for j in range(edge)] + list(range(length - last, length))


def check_evict(hip, ctx, cache, budget, first, last):
    kv, page = cache.k_pages.shape[1], cache.page_size
    lens, slots = ctx.kv_len.tolist(), ctx.state_slots.tolist()
    k, v, w = cache.k_pages.clone(), cache.v_pages.clone(), cache.weights.clone()
    table, host = cache.block_table.long(), cache.weights.double().cpu()
    kept, lengths = hip.evict_cache(ctx, cache, budget, keep_first=first, keep_last=last)
    assert kept.dtype == torch.int32 and kept.shape == (len(lens), kv, budget) and lengths.tolist() == [min(n, budget) for n in lens]
    want_k, want_v, want_w = k.clone(), v.clone(), w.clone()
    for s, length in enumerate(lens):
        n = min(length, budget)
        to = torch.arange(n, device=DEV)
        for g in range(kv):
            lay = layout(host[slots[s], g].tolist(), length, budget, first, last)
            assert kept[s, g].tolist() == lay + [-1] * (budget - n), f"sequence {s} head {g}"
            at = torch.tensor(lay, dtype=torch.long, device=DEV)
            want_k[table[s, to // page], g, to % page] = k[table[s, at // page], g, at % page]
            want_v[table[s, to // page], g, :, to % page] = v[table[s, at // page], g, :, at % page]
            want_w[slots[s], g, :n] = w[slots[s], g, at]
    assert torch.equal(cache.k_pages, want_k) and torch.equal(cache.v_pages, want_v)
    assert torch.equal(torch.nan_to_num(cache.weights, 7.0), torch.nan_to_num(want_w, 7.0))
    return kept, lengths


EVICTIONS = [
    # kv lens, kv, dim, value dim, page size, budget, first, last
    ([2], 1, 16, 16, 16, 1, 0, 0),
    ([40], 2, 64, 64, 16, 39, 1, 4),                       # one place too many
    ([41, 7, 39, 40], 2, 64, 64, 16, 40, 4, 16),           # some have nothing to drop
    ([300], 3, 128, 128, 16, 100, 0, 0),
    ([300], 2, 128, 128, 16, 100, 0, 100),                 # only the last
    ([300], 2, 128, 128, 16, 100, 100, 0),                 # only the first
    ([300, 180], 2, 48, 96, 32, 150, 3, 140),              # the last overlap where they go
    ([1000, 17], 1, 80, 80, 16, 20, 2, 7),                 # nearly all goes
    ([90, 33], 2, 36, 20, 12, 31, 1, 5),                   # nothing in eights, pages of no power of two
    ([50], 2, 5, 3, 4, 21, 0, 9),
    ([5000], 2, 64, 64, 64, 2111, 4, 513),
    ([2600, 2049, 2048], 1, 256, 256, 16, 2048, 4, 1025),
    ([9], 2, 64, 64, 16, 2, 1, 1),                         # nothing between is kept
    ([20000, 700], 1, 16, 16, 64, 9000, 3, 4000),          # more places than a workgroup's registers hold keys of
    ([3000], 1, 8, 8, 1, 1100, 0, 3),                      # a place a page, more pages than LDS holds of the table
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kv_lens,kv,dim,vdim,page,budget,first,last", EVICTIONS)
def test_evict_cache(hip, dtype, kv_lens, kv, dim, vdim, page, budget, first, last):
    slots = torch.randperm(len(kv_lens) + 2, generator=torch.Generator().manual_seed(2)).tolist()[:len(kv_lens)]
    ctx = Ctx([1] * len(kv_lens), kv_lens, slots)
    cache = Cache(kv_lens, kv, page, dim, dtype, value_dim=vdim, n_slots=len(kv_lens) + 2, places=max(kv_lens) + 3)
    check_evict(hip, ctx, cache, budget, first, last)


@pytest.mark.parametrize("kind", ["equal", "few", "zeros", "special", "one bit"])
def test_evict_cache_ties_and_special_weights(hip, kind):
    lens = [1500, 700, 64]
    ctx, cache = Ctx([1] * 3, lens), Cache(lens, 2, 16, 32, torch.bfloat16)
    g = torch.Generator().manual_seed(1)
    shape = cache.weights.shape
    if kind == "equal":
        w = torch.full(shape, 0.75)
    elif kind == "few":
        w = torch.randint(0, 3, shape, generator=g).float()
    elif kind == "zeros":       # both zeros are the same number
        w = torch.where(torch.rand(shape, generator=g) < 0.5, 0.0, -0.0)
    elif kind == "special":
        values = torch.tensor([math.nan, math.inf, -math.inf, 0.0, 1.0, -1.0, 1e-45, 3e38, -math.nan])
        w = values[torch.randint(0, len(values), shape, generator=g)]
    else:                       # neighbours in the last bit: every digit of the key counts
        w = (torch.full(shape, 1.0).view(torch.int32) + torch.randint(0, 5000, shape, generator=g, dtype=torch.int32)).view(torch.float32)
    cache.weights.copy_(w)
    check_evict(hip, ctx, cache, 60, 2, 11)


def test_evict_cache_again_and_again(hip):
    """A token more than the budget at every step, as a server has it: what was moved is right the next time."""
    ctx, cache = Ctx([1], [65]), Cache([65], 2, 16, 64, torch.float32)
    for step in range(8):
        check_evict(hip, ctx, cache, 64, 2, 20)
        cache.weights[:, :, 64] = 0.1 * step
        page = int(cache.block_table[0, 4])
        cache.k_pages[page, :, 0] = rnd(2, 64, seed=step)
        cache.v_pages[page, :, :, 0] = rnd(2, 64, seed=100 + step)


def test_evict_cache_with_bad_pages_and_slots(hip):
    """A page that is none is neither read nor written; a sequence without a row of weights keeps what it has."""
    ctx, cache = Ctx([1, 1], [100, 90], [0, 7]), Cache([100, 90], 1, 16, 32, torch.bfloat16)
    first = cache.block_table[0].clone()
    k = cache.k_pages.clone()
    cache.block_table[0, 1], cache.block_table[0, 3] = -1, cache.k_pages.shape[0]
    kept, _ = hip.evict_cache(ctx, cache, 40, keep_first=1, keep_last=8)
    assert kept[1, 0].tolist() == list(range(40))
    lay = layout(Cache([100, 90], 1, 16, 32, torch.bfloat16).weights[0, 0].tolist(), 100, 40, 1, 8)
    assert kept[0, 0].tolist() == lay
    for i, j in enumerate(lay):
        there, here = int(cache.block_table[0, i // 16]), int(cache.block_table[0, j // 16])
        if i // 16 == 1 or j // 16 in (1, 3):
            assert torch.equal(cache.k_pages[int(first[i // 16]), 0, i % 16], k[int(first[i // 16]), 0, i % 16])
        else:
            assert torch.equal(cache.k_pages[there, 0, i % 16], k[here, 0, j % 16])


def test_evict_cache_of_a_sequence_without_a_row(hip):
    """Its length stays what it was: nothing of it has been dropped."""
    ctx, cache = Ctx([1, 1, 1], [100, 90, 30], [0, 7, -1]), Cache([100, 90, 30], 2, 16, 32, torch.bfloat16)
    k, v, w = cache.k_pages.clone(), cache.v_pages.clone(), cache.weights.clone()
    kept, lengths = hip.evict_cache(ctx, cache, 40, keep_first=1, keep_last=8)
    assert lengths.tolist() == [40, 90, 30]
    assert kept[1, 1].tolist() == list(range(40)) and kept[2, 0].tolist() == list(range(30)) + [-1] * 10
    for s in (1, 2):
        pages = [p for p in cache.block_table[s].tolist() if p >= 0]
        assert torch.equal(cache.k_pages[pages], k[pages]) and torch.equal(cache.v_pages[pages], v[pages])
    assert torch.equal(cache.weights[1:], w[1:])


def test_evict_cache_refuses(hip):
    from simple_inference_amd.kernels import KernelError
    ctx, cache = Ctx([1], [40]), Cache([40], 2, 16, 64, torch.bfloat16)
    k = cache.k_pages.clone()
    for args in ((0,), (-3,), (8, 5, 4), (8, -1), (8, 0, -1), (8, 9)):
        with pytest.raises(KernelError):
            hip.evict_cache(ctx, cache, *args)
    for name, bad in (("k_pages", k.half()), ("k_pages", k[:, :, :8].contiguous()), ("v_pages", k.float()), ("block_table", cache.block_table.long()),
                      ("block_table", cache.block_table[:, :2].contiguous()), ("k_pages", None)):
        own = getattr(cache, name)
        setattr(cache, name, bad)
        with pytest.raises(KernelError):
            hip.evict_cache(ctx, cache, 8)
        setattr(cache, name, own)
    assert torch.equal(cache.k_pages, k)


def test_native_entries_refuse(hip):
    """What the wrappers check first, once more where nothing is launched for it."""
    bad, core, lib = 10001, hip.core, hip._attn_lib(64)
    ctx, cache = Ctx([1], [40]), Cache([40], 2, 16, 64, torch.bfloat16)
    ws, out, ints = torch.zeros(1 << 20, device=DEV), torch.zeros(1 << 16, device=DEV), torch.zeros(1 << 16, dtype=torch.int32, device=DEV)
    k, v, w, t = (x.data_ptr() for x in (cache.k_pages, cache.v_pages, cache.weights, cache.block_table))
    import ctypes

    def rope(counts=(12, 10, 10, 0), axes=3, cycled=0, rows=10, rotary=64, page=16, dtype=1):
        return core.sia_rope_axes_kv_write(out.data_ptr(), 512, ws.data_ptr(), ws.data_ptr(), rows, ints.data_ptr(), (ctypes.c_int * 4)(*counts), axes, cycled,
                                           ctx.positions.data_ptr(), ctx.seq_of_token.data_ptr(), t, 3, k, v, 4, 1, 4, 2, 64, rotary, 0, page, dtype, None)
    for change in (dict(axes=0), dict(axes=5), dict(counts=(12, 10, 9, 0)), dict(counts=(44, -6, -6, 0)), dict(rows=0), dict(rotary=65), dict(rotary=66), dict(page=0),
                   dict(dtype=2), dict(cycled=1, counts=(0, 16, 16, 0))):
        assert rope(**change) == bad

    def evict(budget=8, first=1, last=2, max_kv=40, places=48, ws=ints.data_ptr(), dtype=1, page=16):
        return core.sia_evict(k, v, w, ctx.state_slots.data_ptr(), ctx.kv_len.data_ptr(), t, 3, 4, 1, places, 1, max_kv, 2, 64, 64, page, budget, first, last,
                              ints.data_ptr(), ints.data_ptr(), ws, dtype, None)
    for change in (dict(budget=0), dict(first=-1), dict(last=-1), dict(first=7), dict(max_kv=49), dict(max_kv=60, places=60), dict(places=0), dict(ws=None),
                   dict(dtype=3), dict(page=0)):
        assert evict(**change) == bad

    def attend(lib=lib, single=1, seqs=1, tokens=1, q_bound=0, run_kv=0, max_kv=40, heads=4, kv=2, page=16, scale=0.1, places=48, ws=ws.data_ptr()):
        return lib.sia_attn_weighed(out.data_ptr(), 512, k, v, t, 3, ctx.cu_q.data_ptr(), ctx.kv_len.data_ptr(), out.data_ptr(), ws, single, seqs, tokens, 1, 1, 1,
                                    q_bound, run_kv, max_kv, heads, kv, page, scale, None, w, ctx.state_slots.data_ptr(), 1, places, None)
    for change in (dict(page=12), dict(page=4), dict(heads=5), dict(scale=-1.0), dict(scale=math.nan), dict(places=39), dict(ws=None), dict(max_kv=0), dict(single=2),
                   dict(single=0, tokens=4, q_bound=4, run_kv=41), dict(heads=514, kv=2)):
        assert attend(**change) == bad

    def plain(dim=64, vdim=64, heads=4, q_bound=1, max_kv=40, places=48, ws=ws.data_ptr(), dtype=1):
        return core.sia_attention_weighed(out.data_ptr(), 512, k, v, t, 3, ctx.seq_of_token.data_ptr(), ctx.positions.data_ptr(), ctx.cu_q.data_ptr(),
                                          ctx.kv_len.data_ptr(), out.data_ptr(), ws, 1, 1, 1, q_bound, max_kv, heads, 2, dim, vdim, 16, 4, 0.1, None, w,
                                          ctx.state_slots.data_ptr(), 1, places, dtype, None)
    for change in (dict(dim=0), dict(dim=641), dict(vdim=0), dict(vdim=641), dict(heads=3), dict(q_bound=0), dict(max_kv=49), dict(ws=None), dict(dtype=2)):
        assert plain(**change) == bad


# -- together --------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
def test_a_request_with_a_bounded_cache(hip, dtype):
    """A prompt with a picture in it and some tokens more, the cache cut to its budget whenever it has grown beyond: against a list of
    (key, value, weight) per head that is kept in 64 bits.  What the kernels chose is followed, after a look at whether it may be chosen."""
    heads, kv, dim, budget, first, last, scale = 6, 2, 64, 96, 2, 24, 0.125
    group, sections = heads // kv, (12, 10, 10)
    cache = Cache([256], kv, 16, dim, dtype)
    cache.weights.fill_(math.nan)
    cos, sin = angles(400, 32)
    held = [[] for _ in range(kv)]      # per head: [key, value, weight]
    length = at = 0
    # under a rounding of both sides' keys, values and results, relative to sums of the values' sizes; weights as in check_weighed
    half = torch.finfo(dtype).eps / 2
    for n in [150] + [1] * 10 + [30] + [1] * 5:
        token = torch.arange(at, at + n, dtype=torch.int32)
        where = torch.stack([token, torch.where((token > 20) & (token < 120), 20 + (token - 20) // 10, token),
                             torch.where((token > 20) & (token < 120), 20 + (token - 20) % 10, token)]).to(DEV)
        at += n
        length += n
        ctx = Ctx([n], [length])
        qkv = rnd(n, (heads + 2 * kv) * dim, dtype=dtype, seed=at)
        turned, _ = rotated(qkv, heads + kv, dim, sections, cos, sin, where, "blocks", "half")
        values = qkv[:, (heads + kv) * dim:].double().view(n, kv, dim)
        hip.rope_axes_kv_write(qkv, heads, kv, dim, sections, cos, sin, where, ctx, cache)
        turned = turned.to(dtype).double()
        out = hip.weighed_attention(qkv, heads, kv, dim, scale, ctx, cache).double().view(n, heads, dim)
        for g in range(kv):
            held[g] += [[turned[t, heads + g], values[t, g], 0.0] for t in range(n)]
            k, v = torch.stack([e[0] for e in held[g]]), torch.stack([e[1] for e in held[g]])
            grown = torch.tensor([e[2] for e in held[g]], dtype=torch.float64, device=DEV)
            for h in range(g * group, (g + 1) * group):
                o, p, terms = attended(turned[:, h], k, v, length - n, scale, None)
                # scores: 2 roundings of q and k (their own step each way) beside the float arithmetic
                rel = float(2 * terms * 2 * half + 2 * (dim + 8) * terms * STEP32 + (length + 160) * STEP32)
                assert ((out[:, h] - o).abs() <= half * o.abs() + (p @ v.abs()) * (2 * rel + 1.01 * half)).all()
                grown += p.sum(0)
            got = cache.weights[0, g, :length].double()
            assert ((got - grown).abs() <= grown * (2 * rel + 0.001) * len(token) + 1e-3).all() if dtype == torch.bfloat16 else torch.allclose(got, grown, rtol=1e-3)
            for e, x in zip(held[g], got.tolist()):
                e[2] = x
        if length > budget:
            kept, lengths = hip.evict_cache(ctx, cache, budget, keep_first=first, keep_last=last)
            for g in range(kv):
                lay = layout([e[2] for e in held[g]], length, budget, first, last)
                assert kept[0, g].tolist() == lay
                held[g] = [held[g][j] for j in lay]
            length = int(lengths[0])


def test_a_bounded_cache_in_the_cache_managers_pages(hip):
    """Two requests whose caches are cut to a budget, in pages that the cache manager hands out: pages that one gives back the other writes into, and
    both get the bits that they get alone in pages of their own."""
    from simple_inference_amd.cache import CacheManager
    from simple_inference_amd.parts.context import LayerCache
    from simple_inference_amd.parts.model import CacheLayout
    from simple_inference_amd.parts.plan import PagedKVNeed
    heads, kv, dim, page, budget = 4, 2, 64, 16, 64
    cos, sin = angles(500, 32)
    portions = {0: [100, 1, 1, 40, 1, 1, 1], 1: [30, 50, 1, 1, 60, 1, 1]}

    def serve(requests):
        layout = CacheLayout([PagedKVNeed(kv, dim, None)], [1], [(0, 0)], [], [None])
        books = CacheManager(layout, page_size=page, num_pages=16, max_running=2, dtype=torch.bfloat16, device=DEV)
        weights = torch.full((3, kv, 256), math.nan, device=DEV)
        at, outs = {r: 0 for r in requests}, {r: [] for r in requests}
        for r in requests:
            books.admit(r)
        for turn in range(7):
            step = sorted(requests, key=lambda r: portions[r][turn] != 1)      # single tokens first
            q_lens, lens = [portions[r][turn] for r in step], []
            for r, n in zip(step, q_lens):
                lens.append(books.extend(r, n) + n)
            ctx = Ctx(q_lens, lens, [r for r in step])
            tables = [books.table(0, r) for r in step]
            width = max(len(t) for t in tables)
            table = torch.tensor([t + [-1] * (width - len(t)) for t in tables], dtype=torch.int32, device=DEV)
            layer = books.layer_caches([table])[0]
            assert isinstance(layer, LayerCache) and layer.weights is None
            layer.weights = weights
            rows, where = [], []
            for r, n in zip(step, q_lens):
                rows.append(rnd(n, (heads + 2 * kv) * dim, dtype=torch.bfloat16, seed=1000 * r + at[r]))
                t = torch.arange(at[r], at[r] + n, dtype=torch.int32)
                where.append(torch.stack([t, t // 2, t // 3]))
                at[r] += n
            qkv, where = torch.cat(rows), torch.cat(where, 1).to(DEV).contiguous()
            hip.rope_axes_kv_write(qkv, heads, kv, dim, (12, 10, 10), cos, sin, where, ctx, layer)
            out = hip.weighed_attention(qkv, heads, kv, dim, 0.125, ctx, layer)
            kept, _ = hip.evict_cache(ctx, layer, budget, keep_first=2, keep_last=16)
            for s, (r, length) in enumerate(zip(step, lens)):
                outs[r].append((out[ctx.cu_q[s]:ctx.cu_q[s + 1]].clone(), kept[s].clone()))
                if length > budget:
                    assert books.owns_pages(r)
                    books.shrink(r, budget)
            books.check()
        return outs

    both = serve([0, 1])
    for r in (0, 1):
        for (out, kept), (want, want_kept) in zip(both[r], serve([r])[r]):
            # a run of tokens beside another may take another shape of workgroup: its last bits, and ties of its sums, are its own
            if len(out) == 1:
                assert torch.equal(kept, want_kept)
            torch.testing.assert_close(out.float(), want.float(), rtol=2 ** -7, atol=2 ** -7)


def test_three_operators_in_a_graph(hip):
    """Captured and replayed with eager work between the replays: every replay gives what eager calls give."""
    heads, kv, dim, lens = 8, 2, 64, [700, 130, 65]
    ctx = Ctx([1] * 3, lens, kv_bound=1024)
    cache = Cache(lens, kv, 16, dim, torch.bfloat16, places=1024)
    table = torch.full((3, 64), -1, dtype=torch.int32, device=DEV)
    table[:, :cache.block_table.shape[1]] = cache.block_table
    cache.block_table = table
    cos, sin = angles(900, 32)
    where = torch.zeros(3, 3, dtype=torch.int32, device=DEV)
    qkv = torch.zeros(3, (heads + 2 * kv) * dim, dtype=torch.bfloat16, device=DEV)
    state = [cache.k_pages, cache.v_pages, cache.weights]
    start = [t.clone() for t in state]

    def step():
        hip.rope_axes_kv_write(qkv, heads, kv, dim, (12, 10, 10), cos, sin, where, ctx, cache, order="cycled", pairing="interleaved")
        out = hip.weighed_attention(qkv, heads, kv, dim, 0.125, ctx, cache)
        return (out, *hip.evict_cache(ctx, cache, 64, keep_first=1, keep_last=9))

    def reset(seed):
        for t, s in zip(state, start):
            t.copy_(s)
        qkv.copy_(rnd(*qkv.shape, dtype=torch.bfloat16, seed=seed))
        where.copy_(torch.randint(0, 900, (3, 3), generator=torch.Generator().manual_seed(seed), dtype=torch.int32))

    reset(0)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in range(4):
        reset(seed)
        want = [t.clone() for t in step()] + [t.clone() for t in state]
        torch.cuda.synchronize()
        reset(seed)
        graph.replay()
        for a, b in zip([*got, *state], want):
            assert torch.equal(a, b)


def test_two_graphs_and_two_streams_at_once(hip):
    """Workspaces belong to the call: graphs replayed in turn and streams that run at the same time do not meet."""
    cases = []
    for n, (q_lens, lens) in enumerate((([1] * 4, [1500, 900, 1100, 40]), ([1, 90], [700, 400]))):
        ctx, cache = Ctx(q_lens, lens), Cache(lens, 2, 16, 64, torch.bfloat16, seed=10 * n)
        qkv = rnd(ctx.n_tokens, 8 * 64, dtype=torch.bfloat16, seed=n)
        start = [t.clone() for t in (cache.k_pages, cache.v_pages, cache.weights)]

        def step(ctx=ctx, cache=cache, qkv=qkv):
            out = hip.weighed_attention(qkv, 4, 2, 64, 0.125, ctx, cache)
            return [out, *hip.evict_cache(ctx, cache, 300, keep_first=2, keep_last=50), cache.k_pages, cache.v_pages, cache.weights]

        def reset(cache=cache, start=start):
            for t, x in zip((cache.k_pages, cache.v_pages, cache.weights), start):
                t.copy_(x)

        want = [t.clone() for t in step()]
        reset()
        cases.append((step, reset, want))
    graphs = []
    for step, reset, _ in cases:
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        graphs.append((graph, got))
        reset()
    for _ in range(3):
        for (graph, got), (step, reset, want) in zip(graphs, cases):
            reset()
            graph.replay()
            for a, b in zip(got, want):
                assert torch.equal(a, b)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        results = []
        for stream, (step, reset, _) in zip(streams, cases):
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                reset()
                results.append(step())
        torch.cuda.synchronize()
        for got, (_, _, want) in zip(results, cases):
            for a, b in zip(got, want):
                assert torch.equal(a, b)


def test_pages_beyond_32_bits(hip):
    """A pool whose last pages lie more than 2^32 bytes, and 2^31 elements, behind the first."""
    kv, dim, page = 2, 256, 16
    n_pages = (1 << 31) // (kv * dim * page) + 40
    lens, ctx = [300, 77], Ctx([1, 77], [300, 77])
    cache = Cache(lens, kv, page, dim, torch.bfloat16)
    small, far = (cache.k_pages, cache.v_pages, cache.block_table), n_pages - cache.k_pages.shape[0]
    big_k = torch.empty(n_pages, kv, page, dim, dtype=torch.bfloat16, device=DEV)
    big_v = torch.empty(n_pages, kv, dim, page, dtype=torch.bfloat16, device=DEV)
    big_k[far:], big_v[far:] = small[0], small[1]
    cos, sin = angles(300, 128)
    qkv, weights = rnd(78, 8 * dim, dtype=torch.bfloat16, seed=3), cache.weights.clone()
    where = ctx.positions[None].contiguous()

    def step(rows):
        hip.rope_axes_kv_write(rows, 4, kv, dim, (128,), cos, sin, where, ctx, cache)
        return hip.weighed_attention(rows, 4, kv, dim, 0.0625, ctx, cache), *hip.evict_cache(ctx, cache, 50, keep_last=9), cache.weights

    want = [t.clone() for t in step(qkv.clone())]
    cache.weights.copy_(weights)
    k, v = small[0].clone(), small[1].clone()
    cache.k_pages, cache.v_pages = big_k, big_v
    cache.block_table = torch.where(small[2] >= 0, small[2] + far, small[2])
    for a, b in zip(step(qkv.clone()), want):
        assert torch.equal(a, b)
    assert torch.equal(big_k[far:], k) and torch.equal(big_v[far:], v)


def test_on_a_stream_of_its_own(hip):
    lens = [300, 40]
    ctx, cache = Ctx([1, 40], lens), Cache(lens, 2, 16, 64, torch.bfloat16)
    qkv = rnd(41, 8 * 64, dtype=torch.bfloat16, seed=1)
    start = [t.clone() for t in (cache.weights, cache.k_pages, cache.v_pages)]
    want = hip.weighed_attention(qkv, 4, 2, 64, 0.125, ctx, cache)
    want = [want, *hip.evict_cache(ctx, cache, 30, keep_last=5), cache.weights.clone(), cache.k_pages.clone()]
    cache.weights.copy_(start[0])
    cache.k_pages.copy_(start[1])
    cache.v_pages.copy_(start[2])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = hip.weighed_attention(qkv, 4, 2, 64, 0.125, ctx, cache)
        kept, lengths = hip.evict_cache(ctx, cache, 30, keep_last=5)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip((out, kept, lengths, cache.weights, cache.k_pages), want):
        assert torch.equal(a, b)
