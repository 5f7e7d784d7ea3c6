"""Graphs of the 8-bit cache's operators and of the verification of drafts, several
of them at a time: their workspaces are their own."""

from __future__ import annotations

import pytest
import torch

from light_vllm_b200 import _native, kv8_attention, verify_drafts
from test_kv8_streams_gpu import BATCHES, _Call, _equal

pytestmark = pytest.mark.gpu


def _capture(call, stream):
    """The step as a graph, with no call before it on the stream."""

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = call.run()
    return graph, got


@pytest.mark.parametrize("batch", BATCHES)
def test_graphs_of_one_stream_replayed_side_by_side(batch):
    calls = [_Call(BATCHES[batch], torch.int8, 10 + i) for i in range(3)]
    want = [c.run() for c in calls]
    home = torch.cuda.Stream()
    for c in calls:
        c.reset()
    made = [_capture(c, home) for c in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(30):
        for c, s, (graph, _) in zip(calls, streams, made):
            with torch.cuda.stream(s):
                c.reset()
                graph.replay()
        torch.cuda.synchronize()
        assert all(_equal(got, w) for (_, got), w in zip(made, want))
    assert _native.device_error() == 0


@pytest.mark.parametrize("batch", BATCHES)
def test_a_replay_beside_calls_on_the_capturing_stream(batch):
    calls = [_Call(BATCHES[batch], torch.int8, 20 + i) for i in range(2)]
    want = [c.run() for c in calls]
    home, away = torch.cuda.Stream(), torch.cuda.Stream()
    calls[0].reset()
    graph, got = _capture(calls[0], home)
    for _ in range(30):
        with torch.cuda.stream(away):
            calls[0].reset()
            graph.replay()
        with torch.cuda.stream(home):
            calls[1].reset()
            mine = calls[1].run()
        torch.cuda.synchronize()
        assert _equal(got, want[0]) and _equal(mine, want[1])
    assert _native.device_error() == 0


def test_calls_of_growing_needs_in_one_graph():
    """A decode step, then a prompt's, whose workspace is larger; and more requests to verify."""

    calls = [_Call(BATCHES[b], torch.int8, 30 + i) for i, b in enumerate(("drafts", "prompts", "tokens"))]
    want = [c.run() for c in calls]
    for c in calls:
        c.reset()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):  # torch's own capturing stream
        got = [c.run() for c in calls]
    for _ in range(3):
        for c in calls:
            c.reset()
        graph.replay()
        torch.cuda.synchronize()
        assert all(_equal(g, w) for g, w in zip(got, want))
    assert _native.device_error() == 0


def test_branches_of_one_graph():
    """Attention and verification on two streams that the capture forked to, twice each."""

    calls = [_Call(BATCHES[b], torch.int8, 40 + i) for i, b in enumerate(("tokens", "prompts"))]
    want = [c.run() for c in calls]
    home, side = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()

    def read(c):
        return (kv8_attention(c.rows[:, :8], c.layer, c.step, scale=0.1),
                *verify_drafts(c.probs, c.drafts, c.uniform, c.last, c.step.query_start, max_query_len=c.step.max_query_len))

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=home):
        side.wait_stream(home)
        first = [read(calls[0])]
        with torch.cuda.stream(side):
            second = [read(calls[1]), read(calls[1])]
        first.append(read(calls[0]))
        home.wait_stream(side)
    for _ in range(20):
        graph.replay()
    torch.cuda.synchronize()
    assert all(_equal(g, want[0]) for g in first) and all(_equal(g, want[1]) for g in second)
    assert _native.device_error() == 0
