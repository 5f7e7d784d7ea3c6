"""What the drafting example's command line takes (CPU only)."""

from __future__ import annotations

from types import SimpleNamespace

import pytest

from light_vllm_b200 import KV8Cache, KV8CacheConfig
from test_kv8_backend import example


@pytest.mark.parametrize("requests,drafts", [(1, 0), (4, 7), (12, 7), (64, 7), (1, 300)])
def test_the_runner_holds_every_step(requests, drafts):
    run = example()
    prompts = run.demo_prompts(requests)
    assert len(prompts) == requests and all(0 <= t < 512 for p in prompts for t in p)
    tokens = run.step_tokens(prompts, drafts)
    assert tokens >= sum(map(len, prompts)) and tokens >= requests * (drafts + 1)


def test_more_positions_than_the_model_has():
    run = example()
    runner = SimpleNamespace(device="cpu", shape=SimpleNamespace(max_position_embeddings=64))
    cache = KV8Cache([("a", 4, 2, 64)], KV8CacheConfig(64, 16, device="cpu"))
    with pytest.raises(ValueError, match="64 positions"):
        run.generate(runner, cache, [[1] * 10, [2] * 40], 26, max_drafts=3, temperature=0.0)
