"""The 8-bit cache behind the attention-context contract, and the path that
appends, attends and verifies together.

The tolerances of the whole-model checks: a code is off by a step's uniform
rounding error.  int8: step = block's largest / 127, the largest of some
thousand values is about 3.4 of their standard deviation, so 3.4 / 127 / sqrt(12)
= 0.8 % of a K or V entry's size; e4m3: relative 2^-4 at most, 2^-4 / sqrt(3) / 1.4
= 2.6 %.  A score's error is that share of the score's spread and enters the
weights, a value's enters the output, so an attention output is off by some two
to three of these shares; two layers' add up in the residual: 5 shares with all
of it aligned, 8 with room for rows of few positions, where nothing averages.
"""

from __future__ import annotations

import json
from pathlib import Path

import numpy as np
import pytest
import torch

from light_vllm_b200 import (B200KV8AttentionBackend, B200PagedAttentionBackend, KV8Cache, KV8CacheConfig, KVCacheError, _native,
                             kv8_append, kv8_attention)
from oracle.paged_cache import model_spec, reference_types
from test_kv8_backend import example

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
REF = reference_types()
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
SHARE = {"int8": 8 * 0.008, "e4m3": 8 * 0.026}
GOLDEN = Path(__file__).resolve().parent / "golden" / "qwen2_greedy.npz"


def _metadata(tables, computed, lengths, block):
    used = tuple(tuple(t[:-(-(c + n) // block)]) for t, c, n in zip(tables, computed, lengths))
    return REF.PagedAttentionMetadata(block_tables=used, num_computed_tokens=tuple(computed),
                                      query_layouts=tuple(REF.linear_query_layout(n) for n in lengths))


def _rows(tokens, heads, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn((tokens, heads, 64), device=DEV, generator=gen).half()


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("fused", [False, True])
def test_context_runs_the_operators(code, fused):
    """Three steps of three requests: bit-equal to the operators called by hand."""

    cache, other = (KV8Cache([("a", 4, 2, 64)], KV8CacheConfig(16, 16, CODES[code], DEV)) for _ in range(2))
    backend = B200KV8AttentionBackend()
    tables, computed = [[3, 9, 1], [0, 12, 5], [7, 2, 15]], [0, 0, 0]
    gen = torch.Generator(device=DEV).manual_seed(5)
    angle = torch.rand((64, 64), device=DEV, generator=gen) * 6
    cos, sin = angle.cos().half(), angle.sin().half()
    for number, lengths in enumerate(([17, 1, 20], [1, 1, 1], [4, 13, 1])):
        total = sum(lengths)
        q, k, v = (_rows(total, h, 10 * number + i) for i, h in enumerate((4, 2, 2)))
        context = backend.create(cache, _metadata(tables, computed, lengths, 16))
        step, layer = context.step, other.layer("a")
        if fused:
            positions = torch.tensor([c + j for c, n in zip(computed, lengths) for j in range(n)], dtype=torch.int32, device=DEV)
            qkv = torch.cat([q, k, v], dim=1).view(total, -1)
            context.rope_write_kv("a", qkv, 4, 2, positions, cos, sin)
            rows = qkv.view(total, 8, 64)
            got = context.forward("a", rows[:, :4], rows[:, 4:6], rows[:, 6:], scale=0.125, write_kv=False)
            rotated = kv8_append(q, k, v, layer, step, positions=positions, cos=cos, sin=sin)
            assert torch.equal(rows[:, :4], rotated) and torch.equal(rows[:, 4:], torch.cat([k, v], dim=1))
            want = kv8_attention(rotated, layer, step, scale=0.125)
        else:
            got = context.forward("a", q, k, v, scale=0.125)
            kv8_append(None, k, v, layer, step)
            want = kv8_attention(q, layer, step, scale=0.125)
        assert torch.equal(got, want)
        assert context.layer_ids == frozenset("a")
        for x, y in zip(cache.layer("a"), layer):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
        computed = [c + n for c, n in zip(computed, lengths)]
    assert _native.device_error() == 0


def test_context_refusals():
    cache = KV8Cache([("a", 4, 2, 64)], KV8CacheConfig(4, 16, torch.int8, DEV))
    backend = B200KV8AttentionBackend()
    metadata = _metadata([[0]], [0], [3], 16)
    q, k = _rows(3, 4, 0), _rows(3, 2, 1)
    context = backend.create(cache, metadata)
    for args, message in (((q[0], k, k), "three dimensions"), ((q, k[:2], k[:2]), "token dimensions"), ((q, k, k[:2]), "token dimensions"),
                          ((q[:2], k[:2], k[:2]), "token count"), ((q[:, :2], k, k), "query shape"), ((q, k[:, :1], k[:, :1]), "K/V shape")):
        with pytest.raises(KVCacheError, match=message):
            context.forward("a", *args, scale=1.0)
    with pytest.raises(KVCacheError, match="unknown attention layer"):
        context.forward("b", q, k, k, scale=1.0)
    with pytest.raises(KVCacheError, match="heads or tokens"):
        context.rope_write_kv("a", torch.zeros((3, 512), device=DEV).half(), 2, 3, torch.zeros(3, dtype=torch.int32, device=DEV), q, q)
    context.forward("a", q, k, k, scale=1.0)
    with pytest.raises(KVCacheError, match="ran more than once"):
        context.forward("a", q, k, k, scale=1.0)
    tree = REF.PagedAttentionMetadata(block_tables=((0,),), num_computed_tokens=(0,), query_layouts=(REF.QueryLayout((-1, 0, 0)),))
    with pytest.raises(KVCacheError, match="linear query layouts"):
        backend.create(cache, tree)
    with pytest.raises(KVCacheError):
        backend.create(cache, _metadata([[4]], [0], [3], 16))
    assert _native.device_error() == 0


def _model(max_tokens=192):
    from light_vllm_b200.qwen2 import Qwen2AWQRunner, Qwen2Shape, shard_state_dict

    d = np.load(GOLDEN)
    cfg = json.loads(bytes(d["config_json"]).decode())
    weights = {k[2:]: torch.from_numpy(d[k]) for k in d.files if k.startswith("w:")}
    shape = Qwen2Shape.from_mapping(cfg)
    return Qwen2AWQRunner(shape, shard_state_dict(weights, shape, 0, 1), DEV, max_tokens=max_tokens), [
        d["prompt0"].tolist(), d["prompt1"].tolist()]


def _paged_logits(runner, sequence):
    """Logits of every position over the 16-bit cache, one step."""

    blocks = -(-len(sequence) // 16)
    cache = REF.PagedKVCache(model_spec(REF, runner.kv_layers()), REF.PagedKVCacheConfig(blocks, 16, dtype=torch.float16, device=DEV))
    context = B200PagedAttentionBackend().create(cache, _metadata([list(range(blocks))], [0], [len(sequence)], 16))
    positions = torch.arange(len(sequence), dtype=torch.int32, device=DEV)
    return runner.logits(torch.tensor(sequence, device=DEV), positions, context).float()


@pytest.mark.parametrize("code", CODES)
def test_model_over_the_8_bit_cache(code):
    runner, (prompt, _) = _model()
    try:
        sequence = (prompt * 90)[:90]
        want = _paged_logits(runner, sequence)
        cache = KV8Cache(runner.kv_layers(), KV8CacheConfig(8, 16, CODES[code], DEV))
        backend, rows, computed = B200KV8AttentionBackend(), [], 0
        for n in (37, 1, 1, 30, 5, 16):
            context = backend.create(cache, _metadata([list(range(8))], [computed], [n], 16))
            ids = torch.tensor(sequence[computed:computed + n], device=DEV)
            positions = torch.arange(computed, computed + n, dtype=torch.int32, device=DEV)
            rows.append(runner.logits(ids, positions, context).float())
            assert context.layer_ids == frozenset(cache.layer_ids)
            computed += n
        got = torch.cat(rows)
        assert _native.device_error() == 0
        error = ((got - want).norm() / want.norm()).item()
        assert 0 < error <= SHARE[code], error
        # forward is the greedy token of the same logits
        context = backend.create(cache, _metadata([list(range(8))], [computed - 1], [1], 16))
        last = torch.tensor(sequence[-1:], device=DEV), torch.tensor([computed - 1], dtype=torch.int32, device=DEV)
        token = runner.forward(*last, context)
        context = backend.create(cache, _metadata([list(range(8))], [computed - 1], [1], 16))
        logits = runner.logits(*last, context)[0]
        assert (logits.max() - logits[token]).item() <= 2 * 2.0 ** -11 * logits.abs().max().item()
    finally:
        torch.cuda.synchronize()
        runner.close()


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("drafts", [0, 5])
def test_speculative_decoding(code, drafts):
    """At temperature 0 every token is greedy for what precedes it, drafted or not."""

    runner, prompts = _model()
    run = example()
    prompts = [(p * 4)[:20 + r] for r, p in enumerate(prompts)]  # repetitions, so that drafts are found
    try:
        cache = KV8Cache(runner.kv_layers(), KV8CacheConfig(32, 16, CODES[code], DEV))
        tokens, stats = run.generate(runner, cache, prompts, 60, max_drafts=drafts, temperature=0.0)
        assert _native.device_error() == 0
        assert [len(t) for t in tokens] == [len(p) + 60 for p in prompts]
        assert all(t[:len(p)] == p for t, p in zip(tokens, prompts))
        assert stats["accepted"] <= stats["drafted"] and (stats["drafted"] > 0) == (drafts > 0)
        assert stats["steps"] == 60 if drafts == 0 else stats["steps"] <= 60
        for sequence, prompt in zip(tokens, prompts):
            logits = _paged_logits(runner, sequence)[len(prompt) - 1:-1]
            chosen = logits.gather(1, torch.tensor(sequence[len(prompt):], device=DEV)[:, None])[:, 0]
            # two logits' errors, each six times its usual size of three shares
            size = logits.square().mean(dim=1).sqrt() * SHARE[code] * 3 / 8
            assert ((logits.max(dim=1).values - chosen) <= 2 * 6 * size).all()
    finally:
        torch.cuda.synchronize()
        runner.close()


def test_sampled_decoding_repeats_with_its_seed():
    runner, prompts = _model()
    run = example()
    try:
        results = []
        for seed in (1, 1, 2):
            cache = KV8Cache(runner.kv_layers(), KV8CacheConfig(32, 16, torch.int8, DEV))
            results.append(run.generate(runner, cache, prompts, 40, max_drafts=3, temperature=1.0, seed=seed))
        assert results[0] == results[1] and results[0][0] != results[2][0]
        assert all(0 <= t < 512 for t in results[0][0][0])
    finally:
        torch.cuda.synchronize()
        runner.close()
