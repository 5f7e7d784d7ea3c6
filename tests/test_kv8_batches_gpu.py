"""Batches of more requests than the kernels have threads (they scan such a batch
piece by piece), and contexts that end at, before and after a tile's edge.
Tolerances: test_kv8_gpu.py's."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from light_vllm_b200 import kv8_append, kv8_attention
from test_kv8_gpu import DEV, _check_append, _check_attention, _layer, _np, _rows, _step, _tables

pytestmark = pytest.mark.gpu


def _batch(n, queries, longest, seed):
    """Requests of up to ``longest`` tokens, some of them without query tokens, the last with."""

    rng = np.random.default_rng(seed)
    got = [(int(rng.integers(0, longest)), 0 if i % 11 == 5 else int(queries[i % len(queries)])) for i in range(n)]
    return got[:-1] + [(longest, int(max(queries)))]


def _attend(requests, heads, code, dtype, bs=16):
    hq, hkv, d = heads
    tables, blocks = _tables(requests, bs)
    layer = _layer(blocks, hkv, bs, d, code, seed=1)
    gen = torch.Generator(device=DEV).manual_seed(2)
    query = torch.randn((sum(n for _, n in requests), hq, d), device=DEV, generator=gen).to(dtype)
    step = _step(tables, requests)
    out = kv8_attention(query, layer, step, scale=d ** -0.5)
    _check_attention(query, layer, step, tables, requests, code, d ** -0.5, out)


# Threads of a decode CTA: 128 for up to 8 rows, 256 above; of a tile CTA: 416.
@pytest.mark.parametrize("n", [127, 128, 129, 256, 300, 1030])
def test_many_single_tokens(n):
    _attend(_batch(n, [1], 90, n), (7, 1, 64), "int8", torch.float16)


@pytest.mark.parametrize("n", [129, 400])
def test_many_single_tokens_of_longer_contexts(n):
    """Enough pages for equal runs that cross requests."""

    _attend(_batch(n, [1], 900, n), (8, 4, 128), "e4m3", torch.bfloat16)


@pytest.mark.parametrize("n,heads", [(256, (14, 2, 64)), (257, (14, 2, 64)), (300, (7, 1, 128)), (700, (7, 1, 64))], ids=str)
def test_many_requests_with_drafts(n, heads):
    _attend(_batch(n, [5, 1, 3, 9], 120, n), heads, "int8", torch.bfloat16)


@pytest.mark.parametrize("n", [415, 416, 417, 900])
def test_many_chunks(n):
    _attend(_batch(n, [33, 1, 1, 70, 1], 100, n), (2, 1, 64), "e4m3", torch.float16, bs=32)


@pytest.mark.parametrize("n,queries", [(300, [1]), (700, [1, 4, 2])], ids=["tokens", "drafts"])
def test_many_appends(n, queries):
    requests = _batch(n, queries, 60, n)
    tables, blocks = _tables(requests, 16)
    layer = _layer(blocks, 2, 16, 64, "int8", seed=3, size=0.7)
    before = [t.clone() for t in layer]
    _, key, value = _rows(sum(q for _, q in requests), 1, 2, 64, torch.float16, seed=4)
    kv8_append(None, key, value, layer, _step(tables, requests))
    _check_append(before, layer, {"key": _np(key).astype(np.float64), "value": _np(value).astype(np.float64)}, tables, requests,
                  "int8", 16)


@pytest.mark.parametrize("end", [2047, 2048, 2049, 4095, 4096, 4097])
@pytest.mark.parametrize("queries", [1, 5, 130])
@pytest.mark.parametrize("code,bs", [("int8", 16), ("e4m3", 64)])
def test_contexts_that_end_at_an_edge(end, queries, code, bs):
    requests = [(end - queries, queries), (end - 1, 1)]
    _attend(requests, (7, 1, 64), code, torch.float16, bs)


@pytest.mark.parametrize("computed", [2047, 2048, 2049])
@pytest.mark.parametrize("new", [1, 15, 16, 17, 64, 128])
@pytest.mark.parametrize("code,bs", [("int8", 16), ("e4m3", 64)])
def test_appends_at_a_block_edge(computed, new, code, bs):
    requests = [(computed, new), (new, 1)]
    tables, blocks = _tables(requests, bs)
    layer = _layer(blocks, 2, bs, 64, code, seed=5, size=0.7)
    before = [t.clone() for t in layer]
    _, key, value = _rows(new + 1, 1, 2, 64, torch.bfloat16, seed=6)
    kv8_append(None, key, value, layer, _step(tables, requests))
    _check_append(before, layer, {"key": _np(key).astype(np.float64), "value": _np(value).astype(np.float64)}, tables, requests,
                  code, bs)


def test_the_longest_sequence_named_changes_nothing():
    """max_seq_len bounds nothing: the same bits whatever it says."""

    requests = [(2000, 1), (1200, 2), (100, 300)]
    tables, blocks = _tables(requests, 16)
    layer = _layer(blocks, 4, 16, 128, "int8", seed=7)
    query = torch.randn((303, 28, 128), device=DEV).half()
    want = kv8_attention(query, layer, _step(tables, requests), scale=0.1)
    for named in (0, 16, 100000):
        assert torch.equal(kv8_attention(query, layer, _step(tables, requests, max_seq=named), scale=0.1), want)
