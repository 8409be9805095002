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
