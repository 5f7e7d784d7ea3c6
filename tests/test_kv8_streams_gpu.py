"""The 8-bit cache's operators and the verification of drafts in CUDA graphs, on
several streams, and called again: always the same bits."""

from __future__ import annotations

import pytest
import torch

from light_vllm_b200 import KV8Layer, KV8Step, _native, kv8_append, kv8_attention, verify_drafts

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


class _Call:
    """One step's inputs: append, attend, verify."""

    def __init__(self, requests, code, seed, d=64):
        gen = torch.Generator(device=DEV).manual_seed(seed)
        blocks = [-(-(c + n) // 16) for c, n in requests]
        total, width = sum(n for _, n in requests), max(blocks)
        ids = torch.randperm(sum(blocks), device=DEV, generator=gen).int()
        tables = torch.zeros((len(requests), width), dtype=torch.int32, device=DEV)
        at = 0
        for r, b in enumerate(blocks):
            tables[r, :b] = ids[at:at + b]
            at += b
        starts = torch.tensor([sum(n for _, n in requests[:r]) for r in range(len(requests) + 1)], dtype=torch.int32, device=DEV)
        self.step = KV8Step(tables, torch.tensor([c for c, _ in requests], dtype=torch.int32, device=DEV), starts,
                            max(n for _, n in requests), max(c + n for c, n in requests))
        codes = torch.randint(-100, 100, (2, at, 2, 16, d), dtype=torch.int8, device=DEV, generator=gen)
        codes[codes == -1] = 1  # (NaN in e4m3)
        scales = torch.rand((2, at, 2), device=DEV, generator=gen) * 0.02 + 1e-3
        self.layer = KV8Layer(*codes.view(code), *scales)
        self.codes = codes.clone(), scales.clone()
        self.rows = torch.randn((total, 12, d), device=DEV, generator=gen).half()
        self.probs = torch.softmax(torch.randn((total, 5000), device=DEV, generator=gen) * 3, dim=1)
        drafts = total - len(requests)
        self.drafts = torch.randint(0, 5000, (drafts,), device=DEV, generator=gen)
        self.uniform = torch.rand(drafts, device=DEV, generator=gen) * 1e-3
        self.last = torch.rand(len(requests), device=DEV, generator=gen)

    def reset(self):
        self.layer.keys.view(torch.int8).copy_(self.codes[0][0])
        self.layer.values.view(torch.int8).copy_(self.codes[0][1])
        self.layer.key_scales.copy_(self.codes[1][0])
        self.layer.value_scales.copy_(self.codes[1][1])

    def run(self):
        kv8_append(None, self.rows[:, 8:10], self.rows[:, 10:], self.layer, self.step)
        out = kv8_attention(self.rows[:, :8], self.layer, self.step, scale=0.1)
        return (out, *verify_drafts(self.probs, self.drafts, self.uniform, self.last, self.step.query_start,
                                    max_query_len=self.step.max_query_len))


BATCHES = {"tokens": [(900 + 37 * r, 1) for r in range(12)], "drafts": [(1500, 6), (30, 4), (700, 1)],
           "prompts": [(0, 300), (2000, 1), (100, 64)]}


def _equal(got, want):
    return all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("code", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("batch", BATCHES)
def test_calls_repeat_bit_for_bit(batch, code):
    call = _Call(BATCHES[batch], code, 1)
    want = call.run()
    for _ in range(20):
        call.reset()
        assert _equal(call.run(), want)
    assert _native.device_error() == 0


@pytest.mark.parametrize("batch", BATCHES)
def test_captured_graph(batch):
    call, other = _Call(BATCHES[batch], torch.int8, 2), _Call(BATCHES[batch], torch.int8, 3)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        want = call.run()
        call.reset()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = call.run()
    torch.cuda.synchronize()
    for _ in range(3):
        call.reset()
        graph.replay()
        assert _equal(got, want)
    # the same graph over another step's contents
    want = other.run()
    other.reset()
    for mine, theirs in ((call.layer, other.layer), (call.step[:3], other.step[:3])):
        for a, b in zip(mine, theirs):
            a.copy_(b)
    for name in ("rows", "probs", "drafts", "uniform", "last"):
        getattr(call, name).copy_(getattr(other, name))
    graph.replay()
    assert _equal(got, want)
    assert _native.device_error() == 0


def test_streams_side_by_side():
    calls = [_Call(BATCHES[b], torch.int8, 4 + i) for i, b in enumerate(("tokens", "drafts", "prompts", "tokens"))]
    want = [c.run() for c in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    for c in calls:
        c.reset()
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for c, s in zip(calls, streams):
            with torch.cuda.stream(s):
                c.reset()
                got.append(c.run())
        torch.cuda.synchronize()
        assert all(_equal(g, w) for g, w in zip(got, want))
    assert _native.device_error() == 0
