"""The 8-bit cache's objects and the drafting example's host side (CPU only)."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

from light_vllm_b200 import B200KV8AttentionBackend, B200PagedAttentionBackend, KV8Cache, KV8CacheConfig, KVCacheError, compact_kv

LAYERS = (("a", 4, 2, 64), ("b", 8, 1, 128))


def example():
    path = Path(__file__).resolve().parents[1] / "examples" / "speculative_kv8.py"
    spec = importlib.util.spec_from_file_location("speculative_kv8", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("code", [torch.int8, torch.float8_e4m3fn])
def test_cache_geometry(code):
    cache = KV8Cache(LAYERS, KV8CacheConfig(5, 32, code, "cpu"))
    assert cache.layer_ids == ("a", "b")
    layer = cache.layer("b")
    assert layer.keys.shape == layer.values.shape == (5, 1, 32, 128) and layer.keys.dtype == layer.values.dtype == code
    assert layer.key_scales.shape == layer.value_scales.shape == (5, 1) and layer.key_scales.dtype == torch.float32
    assert not any(t.float().any() for t in layer)
    with pytest.raises(KVCacheError, match="unknown attention layer 'c'"):
        cache.layer("c")


@pytest.mark.parametrize("change,message", [
    (dict(num_blocks=0), "num_blocks"), (dict(num_blocks=True), "num_blocks"), (dict(block_size=24), "multiple of 16"),
    (dict(block_size=0), "multiple of 16"), (dict(block_size=2048), "up to 1024"), (dict(dtype=torch.float16), "int8 or float8"),
])
def test_config_refusals(change, message):
    with pytest.raises(ValueError, match=message):
        KV8CacheConfig(**{**dict(num_blocks=4, block_size=16, dtype=torch.int8, device="cpu"), **change})


@pytest.mark.parametrize("layer,message", [(("a", 4, 2, 80), "64 and 128"), (("a", 3, 2, 64), "multiple"), (("a", 4, 0, 64), "multiple")])
def test_layer_refusals(layer, message):
    with pytest.raises(ValueError, match=message):
        KV8Cache([layer], KV8CacheConfig(4, 16, torch.int8, "cpu"))


def test_other_paths_refuse_the_cache_and_the_backend_a_host():
    cache = KV8Cache(LAYERS, KV8CacheConfig(4, 16, torch.int8, "cpu"))
    metadata = example().step_metadata([[0]], [0], [3], 16)
    with pytest.raises(KVCacheError, match="CUDA KV cache"):
        B200KV8AttentionBackend().create(cache, metadata)
    with pytest.raises(KVCacheError, match="CUDA KV cache"):
        B200PagedAttentionBackend().create(cache, metadata)
    with pytest.raises(KVCacheError):
        compact_kv(cache, [0], num_computed_tokens=0, num_query_tokens=3, num_reserved_query_tokens=3,
                   retained_query_indices=[1])


@pytest.mark.parametrize("tokens,count,want", [
    ([1, 2, 3, 1, 2], 2, [3, 1]), ([1, 2, 3, 1, 2], 8, [3, 1, 2]), ([5, 5, 5, 5], 3, [5]), ([1, 2, 9, 1, 2, 8, 1, 2], 1, [8]),
    ([1, 2, 3], 4, []), ([7], 4, []), ([1, 2, 3, 1, 2], 0, []),
])
def test_lookup_drafts(tokens, count, want):
    assert example().lookup_drafts(tokens, count) == want
