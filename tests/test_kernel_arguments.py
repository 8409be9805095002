"""What the kernels' wrappers make of the device and the context they are given, without a GPU: tensors that say that they are on one, and a
library that only counts its calls."""

import types

import pytest
import torch

from simple_inference_amd.kernels import HipKernels, KernelError
from simple_inference_amd.parts.context import LayerCache


class OnGpu(torch.Tensor):
    """A tensor in host memory that says it is on GPU ``index``."""
    index = 0
    is_cuda = property(lambda self: True)

    def get_device(self):
        return self.index


class OnSecondGpu(OnGpu):
    index = 1


def on(t, kind=OnGpu):
    return t.as_subclass(kind)


class Library:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append(name)
            return {"sia_rope_axes_max": 4, "sia_attention_generic_max_head_dim": 640, "sia_attn_prefill_rows": 128}.get(name, 0)
        return call


def kernels(index=0, current=0):
    k = HipKernels.__new__(HipKernels)
    k.core, k.use_mfma_attention, k._axes_known = Library(), False, {}
    k._device_index, k._current_device, k._raw_stream = index, lambda: current, lambda device: device
    return k


def a_step(kind=OnGpu, n=3, heads=4, kv=2, dim=64):
    """A step of one sequence with n tokens, its cache, and the arguments of the three operators."""
    i32 = lambda x: on(torch.tensor(x, dtype=torch.int32), kind)
    ctx = types.SimpleNamespace(
        n_tokens=n, n_seqs=1, positions=i32(list(range(n))), seq_of_token=i32([0] * n), cu_q=i32([0, n]), kv_len=i32([n]), state_slots=i32([0]),
        max_q_len=n, max_kv_len=n, kv_bound=0, n_decode_seqs=0, q_lens=[n], max_run_kv_len=n, max_single_kv_len=0)
    cache = LayerCache(k_pages=on(torch.zeros(2, kv, 16, dim), kind), v_pages=on(torch.zeros(2, kv, dim, 16), kind), block_table=i32([[1]]), page_size=16,
                       weights=on(torch.zeros(1, kv, 16), kind))
    qkv, table = on(torch.zeros(n, (heads + 2 * kv) * dim), kind), on(torch.zeros(8, dim // 2), kind)
    where = on(torch.zeros(2, n, dtype=torch.int32), kind)
    return ctx, cache, {
        "rotate": lambda k: k.rope_axes_kv_write(qkv, heads, kv, dim, (16, 16), table, table, where, ctx, cache),
        "attend": lambda k: k.weighed_attention(qkv, heads, kv, dim, 0.125, ctx, cache),
        "evict": lambda k: k.evict_cache(ctx, cache, 8)}


OPERATORS = ["rotate", "attend", "evict"]
ENTRIES = {"rotate": "sia_rope_axes_kv_write", "attend": "sia_attention_weighed", "evict": "sia_evict"}


@pytest.mark.parametrize("name", OPERATORS)
def test_the_operators_reach_their_kernels(name):
    for index, kind in ((0, OnGpu), (1, OnSecondGpu)):
        k = kernels(index, index)
        a_step(kind)[2][name](k)
        assert k.core.calls[-1] == ENTRIES[name]


@pytest.mark.parametrize("name", OPERATORS)
def test_the_operators_of_a_bounded_cache_refuse_another_device(name):
    for k, kind in ((kernels(0, 0), OnSecondGpu), (kernels(1, 1), OnGpu), (kernels(0, 1), OnGpu)):
        with pytest.raises(KernelError):
            a_step(kind)[2][name](k)
        assert ENTRIES[name] not in k.core.calls


def test_other_kernels_take_what_is_on_a_gpu():
    """As a process has it that made another GPU the current one and runs there on its default stream."""
    k = kernels(0, 1)
    t = on(torch.zeros(4, 8), OnSecondGpu)
    k._want(t, "rows", torch.float32, (4, 8))
    ctx, cache, _ = a_step(OnSecondGpu)
    k._check_pages(cache.k_pages, cache.v_pages, cache.block_table, 16, 2, 64, torch.float32, ctx)
    k.paged_attention(on(torch.zeros(3, 8 * 64), OnSecondGpu), 4, 2, 64, 0.125, None, ctx, cache)
    assert k.core.calls[-1] == "sia_attention_f32"
    for bad in (torch.zeros(4, 8), t.double(), on(torch.zeros(8, 4).t(), OnSecondGpu), on(torch.zeros(4, 9), OnSecondGpu)):
        with pytest.raises(KernelError):
            k._want(bad, "rows", torch.float32, (4, 8))


READ = {"rotate": ["positions", "seq_of_token"], "attend": ["positions", "seq_of_token", "cu_q", "kv_len", "state_slots"], "evict": ["kv_len", "state_slots"]}


@pytest.mark.parametrize("name,field", [(name, field) for name in OPERATORS for field in READ[name]])
def test_what_the_kernels_read_of_a_context_is_checked(name, field):
    for change in (lambda t: on(t.long()), lambda t: on(t[:-1].contiguous()), lambda t: on(torch.cat([t, t])), lambda t: on(t.repeat_interleave(2)[::2]),
                   lambda t: on(t[None]), lambda t: on(t.float()), lambda t: t.as_subclass(torch.Tensor), lambda t: on(t, OnSecondGpu)):
        k, (ctx, _, calls) = kernels(), a_step()
        own, changed = getattr(ctx, field), change(getattr(ctx, field))
        if changed.is_contiguous() and changed.shape == own.shape and changed.dtype == own.dtype and type(changed) is OnGpu:
            continue      # (one number in every other place is one number)
        setattr(ctx, field, changed)
        with pytest.raises(KernelError):
            calls[name](k)
        assert ENTRIES[name] not in k.core.calls


@pytest.mark.parametrize("n_decode", [-1, 2])
def test_single_tokens_that_a_step_has_not(n_decode):
    k, (ctx, _, calls) = kernels(), a_step()
    ctx.n_decode_seqs = n_decode
    with pytest.raises(KernelError):
        calls["attend"](k)
    assert ENTRIES["attend"] not in k.core.calls


def test_a_rotation_without_pages_reads_no_places():
    k, (ctx, _, _) = kernels(), a_step()
    ctx.positions = ctx.seq_of_token = torch.zeros(0)
    qkv, table, where = on(torch.zeros(3, 4 * 64)), on(torch.zeros(8, 32)), on(torch.zeros(2, 3, dtype=torch.int32))
    k.rope_axes_kv_write(qkv, 4, 0, 64, (16, 16), table, table, where, ctx, None)
    assert k.core.calls[-1] == "sia_rope_axes_kv_write"


class Built(Exception):
    pass


def test_the_kernels_are_made_for_the_configured_device(monkeypatch):
    from simple_inference_amd import Engine, EngineConfig
    from simple_inference_amd import kernels as package
    from simple_inference_amd.engine import build

    def made(device="cuda:0"):
        raise Built(device)
    monkeypatch.setattr(package, "HipKernels", made)
    for device, want in (("cuda:1", "cuda:1"), ("cuda:0", "cuda:0"), ("cuda", "cuda"), ("cpu", "cuda:0")):
        cfg = EngineConfig(device=device, max_seq_len=64)
        for call in (lambda: build.default_kernels(device), lambda: Engine.from_folder("nowhere", cfg), lambda: Engine.from_random({}, 0, cfg),
                     lambda: build.model_from_folder("nowhere", cfg), lambda: build.model_from_random({}, 0, cfg)):
            with pytest.raises(Built) as e:
                call()
            assert e.value.args == (want,)
    with pytest.raises(Built) as e:
        build.default_kernels()
    assert e.value.args == ("cuda:0",)
