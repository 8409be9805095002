"""What a step's context says of its sequences' lengths on the host (no GPU)."""

import pytest

from helpers import TINIES, make_runner, random_tokens, write_tiny_model
from simple_inference_amd.engine import StepEntry


@pytest.fixture(scope="module")
def folder(tmp_path_factory):
    return write_tiny_model(tmp_path_factory.mktemp("bounds"), TINIES["b"], seed=3)


def test_longest_single_token_and_longest_run(folder):
    runner, cache, cfg = make_runner(folder, "twins", 8, 64)
    tokens = random_tokens(cfg.vocab_size, 90, seed=1)
    for req in range(4):
        cache.admit(req)
    ctx = runner.build_context([StepEntry(0, tokens[:40]), StepEntry(1, tokens[:9])])
    assert (ctx.max_kv_len, ctx.max_run_kv_len, ctx.max_single_kv_len) == (40, 40, 0)
    ctx = runner.build_context([StepEntry(2, tokens[:70]), StepEntry(0, tokens[:1]), StepEntry(1, tokens[:1]), StepEntry(3, tokens[:1])])
    assert (ctx.n_decode_seqs, ctx.max_kv_len, ctx.max_run_kv_len, ctx.max_single_kv_len) == (3, 70, 70, 41)
    ctx = runner.build_context([StepEntry(2, tokens[:1]), StepEntry(3, tokens[:1])])
    assert (ctx.max_kv_len, ctx.max_run_kv_len, ctx.max_single_kv_len) == (71, 0, 71)
