"""Three operators of a cache that holds less than a request's past, as cases that can be timed.

A long request of text, pictures and video does not keep every token it has read.  Its tokens are rotated by positions
with several axes and written to the next places of their sequence's pages (``rotate``); attention over the pages also
adds up how much weight every cached token got (``attend``); and when a sequence has grown beyond its budget, the tokens
that got least are dropped and the others closed up (``evict``).  After that a token's place in the cache is no longer
its position, which is why the rotation takes positions of its own.

    rotate   q and k of token t, pair j of the rotary ones, turned by the table's angle of position[axis(j), t]:
             a' = a cos - b sin, b' = b cos + a sin; k and v written to place ctx.positions[t]
    attend   p[t, h, j] = exp(s[t, h, j]) / sum_j' exp(s[t, h, j']) over the places j <= ctx.positions[t], s = scale q.k;
             out[t, h] = sum_j p v_j;  weights[slot, g, j] += sum over the sequence's t and the heads h of g of p[t, h, j],
             where the sum of a place that the step itself has written begins at zero
    evict    of every sequence with more than ``budget`` places and for every key/value head: the first ``keep_first``,
             the last ``keep_last``, and of those between the ones with the largest weight (ties: the lowest place).
             The last stay the last; of the others the kept ones below ``budget - keep_last`` stay where they are and
             the kept ones from beyond fill the holes, both in order.  Keys, values and weights move.

A case: ``op``, ``dtype``; ``heads`` on ``kv`` of ``dim``; ``rows`` sequences that bring one token each over about
``context`` tokens (``ragged``: from half to one and a half times as many) and one that brings ``prompt`` tokens over
``past``; ``page`` places a page.  ``rotate``: ``axes`` of positions (with ``cycled``: dealt to the pairs in turn, else in blocks),
``rotary`` rotated elements of a head, ``neighbours``: whether 2i and 2i + 1 make a pair, or i and i + rotary / 2.  ``evict``: ``budget``,
``first`` and ``last``.

``own``: whether ``run`` makes the framework's calls or computes the plain forms.
"""

import math

import torch

own = False

_kernels = None


def _case(op, heads, kv, dim, rows=0, context=0, ragged=False, prompt=0, past=0, dtype="bfloat16", page=16, **more):
    return dict({"op": op, "heads": heads, "kv": kv, "dim": dim, "rows": rows, "context": context, "ragged": ragged, "prompt": prompt,
                 "past": past, "dtype": dtype, "page": page}, **more)


def _rotate(heads, kv, dim, axes=3, cycled=False, rotary=None, neighbours=False, **more):
    return _case("rotate", heads, kv, dim, axes=axes, cycled=cycled, rotary=rotary or dim, neighbours=neighbours, **more)


def _evict(heads, kv, dim, budget, first, last, **more):
    return _case("evict", heads, kv, dim, budget=budget, first=first, last=last, **more)


def listed():
    named = [
        # eight users' next tokens: latency
        ("rotate 8 rows", _rotate(24, 8, 128, rows=8, context=2048, ragged=True)),
        # a prompt with pictures
        ("rotate prompt 2048", _rotate(24, 8, 128, prompt=2048)),
        # some minutes of video in one step, of a size that divides nothing
        ("rotate prompt 16411", _rotate(32, 8, 128, prompt=16411, past=37)),
        # the 32-bit path, a part of every head rotated, axes in turn, a portion beside decoded tokens
        ("rotate float32 303", _rotate(32, 8, 64, axes=2, cycled=True, rotary=48, neighbours=True, rows=3, context=200, ragged=True, prompt=300,
                                       dtype="float32")),
        # one user at the start of a chat: the shortest call there is
        ("attend 1 row of 40", _case("attend", 32, 8, 64, rows=1, context=40)),
        # eight users whose caches have reached a budget of 2,048
        ("attend 8 rows of 2048", _case("attend", 24, 8, 128, rows=8, context=2048)),
        # a few users with long documents: the cache is all that the step reads
        ("attend 3 ragged of 12000", _case("attend", 32, 8, 128, rows=3, context=12000, ragged=True)),
        # a prompt whose tokens' weights are wanted before the first token is decoded
        ("attend prompt 2048", _case("attend", 24, 8, 128, prompt=2048)),
        # trace replay in the 32-bit path: decoded tokens beside a portion
        ("attend float32 3 and 300", _case("attend", 32, 8, 64, rows=3, context=200, ragged=True, prompt=300, dtype="float32")),
        # eight users that have gone 64 tokens beyond a budget of 2,048, a quarter of it the latest
        ("evict 8 rows of 2112", _evict(24, 8, 128, 2048, 4, 512, rows=8, context=2112)),
        # a document that is cut down to the size of a conversation
        ("evict 16384 to 4096", _evict(32, 8, 128, 4096, 4, 512, rows=1, context=16384)),
        # a full server of the 32-bit path
        ("evict float32 64 rows", _evict(32, 8, 64, 509, 1, 100, rows=64, context=700, ragged=True, dtype="float32")),
    ]
    return [dict(c, name=name) for name, c in named]


def draw(rng):
    """A case of one of the kinds above: sizes spread over their logarithm, odd ones as likely as even ones."""
    size = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    op = rng.choice(["rotate", "attend", "attend", "evict"])
    dtype = "float32" if rng.random() < 0.2 else "bfloat16"
    heads, kv, dim = rng.choice([(24, 8, 128), (32, 8, 64), (32, 8, 128), (8, 8, 64), (16, 1, 128), (20, 4, 80), (6, 2, 256)])
    if dtype == "float32" and dim > 128:
        dim = 96
    page = rng.choice([16, 16, 16, 32, 64])
    rows = size(1, 64)
    if op == "rotate":
        axes, rotary = rng.randint(1, 4), dim if rng.random() < 0.7 else dim // 2
        prompt = rng.choice([0, size(2, 12000 if dtype == "bfloat16" else 3000)])
        return _rotate(heads, kv, dim, axes, rng.random() < 0.5, rotary, rng.random() < 0.3, rows=rows if not prompt or rng.random() < 0.3 else 0,
                       context=size(16, 2000), ragged=True, prompt=prompt, past=rng.choice([0, size(1, 2000)]) if prompt else 0, dtype=dtype,
                       page=page)
    if op == "evict":
        context = size(48, min(16000, 60000 // rows))
        budget = max(8, int(context * rng.uniform(0.2, 0.98)))
        last = int(budget * rng.uniform(0.0, 0.6))
        return _evict(heads, kv, dim, budget, rng.choice([0, 1, 4]), last, rows=rows, context=context, ragged=rng.random() < 0.5, dtype=dtype,
                      page=page)
    if rng.random() < 0.4:
        past = rng.choice([0, 0, size(16, 2000)])
        most = 1800 if dtype == "bfloat16" else 500
        return _case("attend", heads, kv, dim, rows=rng.choice([0, min(rows, 8)]), context=size(16, 1500), ragged=True, prompt=size(2, most),
                     past=past, dtype=dtype, page=page)
    return _case("attend", heads, kv, dim, rows=rows, context=size(16, min(16000, (60000 if dtype == "bfloat16" else 12000) // rows)),
                 ragged=rng.random() < 0.7, dtype=dtype, page=page)


# ---------------------------------------------------------------------------------------------------------
# what a program has in hand
# ---------------------------------------------------------------------------------------------------------

class _Step:
    """The fields of a step's context that these operators read."""


class _Cache:
    """The fields of a layer's cache that these operators read."""


def _lengths(case, seed):
    """(tokens that each sequence brings, tokens that it holds with them, the most that it could hold)."""
    gen = torch.Generator()
    gen.manual_seed(7919 * seed + 5)
    held, half = [case["context"]] * case["rows"], max(1, case["context"] // 2)
    if case["ragged"]:
        held = [half + int(torch.randint(0, case["context"] + 1, (1,), generator=gen)) for _ in held]
    brought, most = [1] * len(held), [case["context"] + (half if case["ragged"] else 0)] * len(held)
    if case["prompt"]:
        brought.append(case["prompt"])
        held.append(case["past"] + case["prompt"])
        most.append(held[-1])
    return brought, held, most


def _sections(case):
    """Pairs of each axis: the first takes what an even share leaves."""
    half = case["rotary"] // 2
    share = half // case["axes"]
    return (half - share * (case["axes"] - 1),) + (share,) * (case["axes"] - 1)


def _axis_of_pair(case):
    sections = _sections(case)
    if case["cycled"]:
        n = case["axes"]
        return [j % n if j % n and j < n * sections[j % n] else 0 for j in range(case["rotary"] // 2)]
    return [a for a, count in enumerate(sections) for _ in range(count)]


def prepare(case, seed):
    """A step's context, a layer's pages with what is cached in them, the projected rows, the tables of angles."""
    dev, dtype = "cuda", getattr(torch, case["dtype"])
    gen = torch.Generator(device=dev)
    gen.manual_seed(1000003 * seed + 29)
    normal = lambda *shape: torch.empty(shape, device=dev).normal_(0.0, 1.0, generator=gen)
    brought, held, most = _lengths(case, seed)
    heads, kv, dim, page = case["heads"], case["kv"], case["dim"], case["page"]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    st = _Step()
    st.case = case
    ctx = st.ctx = _Step()
    ctx.n_seqs, ctx.n_tokens, ctx.q_lens = len(held), sum(brought), brought
    ctx.max_q_len, ctx.max_kv_len, ctx.kv_bound = max(brought), max(held), 0
    ctx.n_decode_seqs = sum(q == 1 for q in brought)
    ctx.max_run_kv_len = max([k for q, k in zip(brought, held) if q > 1], default=0)
    q_len, ctx.kv_len = i32(brought), i32(held)
    ctx.cu_q = torch.cat([i32([0]), q_len.cumsum(0).int()])
    ctx.seq_of_token = torch.repeat_interleave(torch.arange(ctx.n_seqs, device=dev), q_len.long()).int()
    token = torch.arange(ctx.n_tokens, device=dev, dtype=torch.int32)
    ctx.positions = (ctx.kv_len - ctx.cu_q[1:])[ctx.seq_of_token.long()] + token
    slots = ctx.n_seqs + 1                                   # one more, that no sequence has
    ctx.state_slots = torch.randperm(slots, generator=gen, device=dev)[:ctx.n_seqs].int()

    cache = st.cache = _Cache()
    cache.page_size, width = page, -(-max(most) // page)
    room = torch.tensor([-(-k // page) for k in most], device=dev)[:, None]
    pages = int(room.sum())
    order = torch.randperm(pages, generator=gen, device=dev).int()
    first, index = room.cumsum(0) - room, torch.arange(width, device=dev)
    cache.block_table = torch.where(index * page < ctx.kv_len[:, None], order[(first + index).clamp(max=pages - 1)], -1).int()
    # A few of the cached tokens draw most of the weight, as they do in trained models: along a direction of a head's own, that
    # all queries share, keys reach by different amounts.  One more page, that no sequence has, for what is written nowhere.
    along = normal(kv, 1, dim)
    reach = 0.25 * normal(pages + 1, kv, page, 1).exp()
    keys = normal(pages + 1, kv, page, dim) + reach * along
    cache.k_pages = keys.to(dtype)
    cache.v_pages = normal(pages + 1, kv, dim, page).to(dtype)
    cache.weights = normal(slots, kv, width * page).mul_(1.5).exp_().mul_(0.01)
    st.qkv = normal(ctx.n_tokens, heads + 2 * kv, dim)
    st.qkv[:, :heads] += 0.5 * along[:, 0].repeat_interleave(heads // kv, 0)
    st.qkv = st.qkv.view(ctx.n_tokens, -1).to(dtype)
    st.scale = dim ** -0.5
    if case["op"] == "evict":       # some tokens have had no weight at all: they tie
        st.given = cache.weights * (torch.rand(cache.weights.shape, generator=gen, device=dev) > 0.1)
    if case["op"] == "rotate":
        half, axes = case["rotary"] // 2, case["axes"]
        # text in front, where all axes run alike, then frames of 24 x 26 patches: time, height and width
        at, text = ctx.positions.long(), 64
        patch = (at - text).clamp(min=0)
        grid = torch.stack([text + patch // 624, text + patch // 26 % 24, text + patch % 26, text + patch // 7])[:axes]
        if axes == 1:
            grid = at[None]
        st.rotary_positions = torch.where(at[None] < text, at[None], grid).int().contiguous()
        frequency = 500000.0 ** (-torch.arange(half, dtype=torch.float64, device=dev) / half)
        angle = torch.outer(torch.arange(int(st.rotary_positions.max()) + 1, dtype=torch.float64, device=dev), frequency)
        st.cos, st.sin = angle.cos().float(), angle.sin().float()
        st.sections = _sections(case)
        st.axis = torch.tensor(_axis_of_pair(case), device=dev)
    return st


# ---------------------------------------------------------------------------------------------------------
# a pass
# ---------------------------------------------------------------------------------------------------------

def _framework():
    global _kernels
    if _kernels is None:
        from simple_inference_amd.kernels import HipKernels

        _kernels = HipKernels()
    return _kernels


def run(state):
    return {"rotate": _run_rotate, "attend": _run_attend, "evict": _run_evict}[state.case["op"]](state)


def _run_rotate(st):
    case, ctx, cache = st.case, st.ctx, st.cache
    if own:
        _framework().rope_axes_kv_write(
            st.qkv, case["heads"], case["kv"], case["dim"], st.sections, st.cos, st.sin, st.rotary_positions, ctx, cache,
            order="cycled" if case["cycled"] else "blocks", pairing="interleaved" if case["neighbours"] else "half")
    else:
        heads, kv, dim, rotary = case["heads"], case["kv"], case["dim"], case["rotary"]
        half = rotary // 2
        x = st.qkv.view(ctx.n_tokens, heads + 2 * kv, dim)
        qk = x[:, :heads + kv].float()
        at = st.rotary_positions.long()[st.axis].t()                                  # [tokens, pairs]
        pair = torch.arange(half, device=at.device)
        c, s = st.cos[at, pair][:, None], st.sin[at, pair][:, None]
        if case["neighbours"]:
            a, b = qk[..., 0:rotary:2], qk[..., 1:rotary:2]
            turned = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
        else:
            a, b = qk[..., :half], qk[..., half:rotary]
            turned = torch.cat([a * c - b * s, b * c + a * s], -1)
        qk = torch.cat([turned, qk[..., rotary:]], -1).to(st.qkv.dtype)
        x[:, :heads] = qk[:, :heads]
        place = ctx.positions.long()
        page = cache.block_table[ctx.seq_of_token.long(), place // cache.page_size].long()
        cache.k_pages[page, :, place % cache.page_size] = qk[:, heads:]
        cache.v_pages[page, :, :, place % cache.page_size] = x[:, heads + kv:]
    return {"qkv": st.qkv, "keys": cache.k_pages, "values": cache.v_pages}


def _pages_as_rows(cache, dim):
    """Keys and values of all places of every sequence, in 32 bits: [sequences, key/value heads, places, dim]."""
    table = cache.block_table.long().clamp(min=0)
    n, width = table.shape
    k = cache.k_pages[table].transpose(1, 2).reshape(n, -1, width * cache.page_size, dim).float()
    v = cache.v_pages[table].permute(0, 2, 1, 4, 3).reshape(n, -1, width * cache.page_size, dim).float()
    return k, v


def _run_attend(st):
    case, ctx, cache = st.case, st.ctx, st.cache
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    if own:
        out = _framework().weighed_attention(st.qkv, heads, kv, dim, st.scale, ctx, cache)
        return {"out": out, "weights": cache.weights}
    k, v = _pages_as_rows(cache, dim)
    n, most, places = ctx.n_seqs, ctx.max_q_len, k.shape[2]
    slots, length, first = ctx.state_slots.long(), ctx.kv_len.long(), ctx.cu_q.long()
    q_len = first[1:] - first[:-1]
    i, j = torch.arange(most, device=k.device), torch.arange(places, device=k.device)
    row = (first[:-1, None] + i).clamp(max=ctx.n_tokens - 1)                             # [sequences, rows]
    q = st.qkv[row].view(n, most, -1, dim)[:, :, :heads].float()
    q = q.view(n, most, kv, heads // kv, dim).permute(0, 2, 3, 1, 4).reshape(n, kv, -1, dim)
    s = torch.matmul(q, k.transpose(-1, -2)).view(n, kv, heads // kv, most, places) * st.scale
    seen = j <= ((length - q_len)[:, None] + i)[..., None]                               # [sequences, rows, places]
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    e = (s - s.amax(-1, keepdim=True)).exp()
    p = e / e.sum(-1, keepdim=True)
    o = torch.matmul(p.view(n, kv, -1, places), v).view(n, kv, heads // kv, most, dim).permute(0, 3, 1, 2, 4)
    out = o[ctx.seq_of_token.long(), torch.arange(ctx.n_tokens, device=k.device) - first[ctx.seq_of_token.long()]]
    brings = (i < q_len[:, None])[:, None, None, :, None]
    add = (p * brings).sum((2, 3))                                                       # [sequences, key/value heads, places]
    old = cache.weights[slots]
    now = torch.where((j < (length - q_len)[:, None])[:, None], old, torch.zeros_like(old)) + add
    cache.weights[slots] = torch.where((j < length[:, None])[:, None], now, old)
    return {"out": out.reshape(ctx.n_tokens, -1).to(st.qkv.dtype), "weights": cache.weights}


def _run_evict(st):
    case, ctx, cache = st.case, st.ctx, st.cache
    budget, first, last = case["budget"], case["first"], case["last"]
    cache.weights.copy_(st.given)       # a pass moves the weights: the next one has them as they were
    if own:
        kept, lengths = _framework().evict_cache(ctx, cache, budget, keep_first=first, keep_last=last)
    else:
        kept, lengths = _plain_eviction(case, ctx, cache)
    return {"kept": kept, "lengths": lengths, "keys": cache.k_pages[:-1], "values": cache.v_pages[:-1], "weights": cache.weights}


def _plain_eviction(case, ctx, cache):
    budget, first, last = case["budget"], case["first"], case["last"]
    slots, length, page = ctx.state_slots.long(), ctx.kv_len.long()[:, None, None], cache.page_size
    w = cache.weights[slots]                                                             # [sequences, key/value heads, places]
    n, kv, places = w.shape
    j = torch.arange(places, device=w.device).expand(n, kv, places)
    w = torch.where(w.isnan(), torch.full_like(w, -math.inf), w)
    over = length > budget
    # in order of choice: the first and the last, then the others by weight, then what is no place of the sequence
    kind = torch.where((j < first) | (j >= length - last), 0, 1)
    kind = torch.where(j < length, kind, 2)
    choice = w.sort(dim=-1, descending=True, stable=True).indices
    choice = choice.gather(-1, kind.gather(-1, choice).sort(dim=-1, stable=True).indices)
    rank = torch.empty_like(choice).scatter_(-1, choice, j)
    keep = rank < torch.minimum(length, torch.full_like(length, budget))
    # where they go: below the edge they stay, the last move up together, the others fill the holes
    edge = torch.where(over, budget - last, places)
    latest = over & (j >= length - last) & (j < length)
    hole, mover = ~keep & (j < edge), keep & (j >= edge) & ~latest
    holes = torch.zeros(n, kv, places + 1, dtype=torch.long, device=w.device)
    holes.scatter_(-1, torch.where(hole, hole.cumsum(-1) - 1, places), j)
    to = torch.where(mover, holes.gather(-1, (mover.cumsum(-1) - 1).clamp(min=0)), j)
    to = torch.where(latest, j - (length - budget), to)
    kept = torch.full((n, kv, max(budget, places) + 1), -1, dtype=torch.long, device=w.device)
    kept.scatter_(-1, torch.where(keep, to, kept.shape[-1] - 1), j)
    kept = kept[..., :budget]
    # the rows, all read before any is written; what is no row goes to the page that nobody has
    table, g = cache.block_table.long(), torch.arange(kv, device=w.device)[None, :, None]
    seq, i = torch.arange(n, device=w.device)[:, None, None], torch.arange(budget, device=w.device)
    from_ = kept.clamp(min=0)
    here, there = table[seq, from_ // page], table[seq, (i // page).clamp(max=table.shape[1] - 1)]
    there = torch.where(kept >= 0, there, cache.k_pages.shape[0] - 1)
    rows, columns = cache.k_pages[here, g, from_ % page], cache.v_pages[here, g, :, from_ % page]
    cache.k_pages[there, g, i % page] = rows
    cache.v_pages[there, g, :, i % page] = columns
    held = min(budget, places)
    old = cache.weights[slots]
    old[..., :held] = torch.where(kept[..., :held] >= 0, old.gather(-1, from_[..., :held]), old[..., :held])
    cache.weights[slots] = old
    return kept.int(), length[:, 0, 0].clamp(max=budget).int()


# ---------------------------------------------------------------------------------------------------------
# what a pass cannot do without, and what it should give
# ---------------------------------------------------------------------------------------------------------

def work(case):
    """Inputs once, outputs once.  Lengths that go by the seed are taken at their middle."""
    brought, held = [1] * case["rows"], [case["context"]] * case["rows"]
    if case["prompt"]:
        brought, held = brought + [case["prompt"]], held + [case["past"] + case["prompt"]]
    heads, kv, dim, size = case["heads"], case["kv"], case["dim"], 2 if case["dtype"] == "bfloat16" else 4
    n = sum(brought)
    if case["op"] == "rotate":
        # q there and back, k and v there and into the pages, the angles
        return {"bytes": n * (2 * (heads + 2 * kv) * dim * size + 4 * case["rotary"]), "flops": 3 * n * (heads + kv) * case["rotary"]}
    if case["op"] == "attend":
        cached = sum(held)
        seen = sum(q * (k - q) + q * (q + 1) // 2 for q, k in zip(brought, held))
        return {"bytes": cached * kv * (2 * dim * size + 8) + 2 * n * heads * dim * size, "flops": 4 * seen * heads * dim}
    # the weights once; what is kept but beyond the edge is read and written (of those between, as many as an even choice brings there)
    moved = 0.0
    for k in held:
        if k > case["budget"]:
            between, edge = k - case["first"] - case["last"], case["budget"] - case["last"]
            share = (edge - case["first"]) / max(1, between)
            moved += case["last"] + share * max(0, k - case["last"] - edge)
    return {"bytes": sum(held) * kv * 4 + moved * kv * 2 * (2 * dim * size + 4) + 4 * case["budget"] * len(held) * kv, "flops": 0}


def exact(case, seed):
    st = prepare(case, seed)
    return {"rotate": _exact_rotate, "attend": _exact_attend, "evict": _exact_evict}[case["op"]](st)


def _exact_rotate(st):
    """Every token's pairs as complex numbers."""
    case, ctx, cache = st.case, st.ctx, st.cache
    heads, kv, dim, half = case["heads"], case["kv"], case["dim"], case["rotary"] // 2
    qkv = st.qkv.double().view(ctx.n_tokens, heads + 2 * kv, dim).clone()
    first = torch.arange(half, device="cuda") * (2 if case["neighbours"] else 1)
    second = first + (1 if case["neighbours"] else half)
    turn = torch.empty(ctx.n_tokens, half, dtype=torch.complex128, device="cuda")
    for pair, axis in enumerate(_axis_of_pair(case)):
        at = st.rotary_positions[axis].long()
        turn[:, pair] = torch.complex(st.cos[at, pair].double(), st.sin[at, pair].double())
    z = torch.complex(qkv[:, :heads + kv][..., first], qkv[:, :heads + kv][..., second]) * turn[:, None]
    qkv[:, :heads + kv][..., first], qkv[:, :heads + kv][..., second] = z.real, z.imag
    keys, values = cache.k_pages.double(), cache.v_pages.double()
    for s in range(ctx.n_seqs):
        rows = torch.arange(int(ctx.cu_q[s]), int(ctx.cu_q[s + 1]), device="cuda")
        at = int(ctx.kv_len[s]) - len(rows) + torch.arange(len(rows), device="cuda")
        page, off = cache.block_table[s].long()[at // case["page"]], at % case["page"]
        keys[page, :, off] = qkv[rows, heads:heads + kv]
        values[page, :, :, off] = qkv[rows, heads + kv:]
    out = st.qkv.double().view_as(qkv).clone()
    out[:, :heads] = qkv[:, :heads]
    return {"qkv": out.view(ctx.n_tokens, -1), "keys": keys, "values": values}


def _exact_attend(st):
    """Sequence after sequence, head after head."""
    case, ctx, cache = st.case, st.ctx, st.cache
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    q = st.qkv.double().view(ctx.n_tokens, -1, dim)
    out = torch.empty(ctx.n_tokens, heads, dim, dtype=torch.float64, device="cuda")
    weights = cache.weights.double()
    for s in range(ctx.n_seqs):
        lo, hi, length, slot = int(ctx.cu_q[s]), int(ctx.cu_q[s + 1]), int(ctx.kv_len[s]), int(ctx.state_slots[s])
        pages = cache.block_table[s, :-(-length // case["page"])].long()
        start = length - (hi - lo)
        weights[slot, :, start:length] = 0.0
        mask = torch.ones(hi - lo, length, dtype=torch.bool, device="cuda").tril(start)
        for h in range(heads):
            g = h // (heads // kv)
            k = cache.k_pages[pages, g].double().reshape(-1, dim)[:length]
            v = cache.v_pages[pages, g].double().transpose(1, 2).reshape(-1, dim)[:length]
            logits = (q[lo:hi, h] @ k.t() * st.scale).masked_fill(~mask, -math.inf)
            p = torch.softmax(logits, -1)
            out[lo:hi, h] = p @ v
            weights[slot, g, :length] += p.sum(0)
    return {"out": out.view(ctx.n_tokens, -1), "weights": weights}


def _exact_evict(st):
    """Head after head on the host: places sorted as Python sorts."""
    import numpy as np

    case, ctx, cache = st.case, st.ctx, st.cache
    kv, budget, first, last, page = case["kv"], case["budget"], case["first"], case["last"], case["page"]
    given = st.given.cpu().numpy()
    moved = given.astype(np.float64)
    kept = np.full((ctx.n_seqs, kv, budget), -1, dtype=np.int64)
    lengths = ctx.kv_len.cpu().numpy()
    for s in range(ctx.n_seqs):
        length, slot = int(lengths[s]), int(ctx.state_slots[s])
        for g in range(kv):
            if length <= budget:
                kept[s, g, :length] = np.arange(length)
                continue
            w = given[slot, g, :length]
            between = np.arange(first, length - last)
            best = between[np.lexsort((between, -w[between]))][:budget - first - last]
            body = np.sort(np.concatenate([np.arange(first), best]))
            edge = budget - last
            lay = np.full(edge, -1)
            stay = body[body < edge]
            lay[stay] = stay
            lay[lay < 0] = body[body >= edge]
            kept[s, g] = np.concatenate([lay, np.arange(length - last, length)])
            moved[slot, g, :budget] = w[kept[s, g]]
    keys, values = cache.k_pages.clone(), cache.v_pages.clone()
    table = cache.block_table.long()
    for s in range(ctx.n_seqs):
        n = min(int(lengths[s]), budget)
        to = torch.arange(n, device="cuda")
        there = table[s, to // page]
        for g in range(kv):
            at = torch.from_numpy(kept[s, g, :n]).cuda()
            here = table[s, at // page]
            keys[there, g, to % page] = cache.k_pages[here, g, at % page]
            values[there, g, :, to % page] = cache.v_pages[here, g, :, at % page]
    return {"kept": torch.from_numpy(kept.astype(np.int32)), "lengths": torch.from_numpy(np.minimum(lengths, budget)),
            "keys": keys[:-1].double(), "values": values[:-1].double(), "weights": torch.from_numpy(moved)}
