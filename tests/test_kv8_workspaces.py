"""Whose scratch a call gets: a stream's, or the graph's that it is captured into (CPU only)."""

from __future__ import annotations

import pytest
import torch

from light_vllm_b200 import _native
from light_vllm_b200.kv8 import _Workspaces

HOST = torch.device("cpu", 0)


class _NoModule:
    def set_scratch(self, *args):
        pass


@pytest.fixture
def capture(monkeypatch):
    current = {"id": 0}
    monkeypatch.setattr(_native, "stream_capture_id", lambda stream: current["id"], raising=False)
    monkeypatch.setattr(_native, "torch_ops", _NoModule)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: bool(current["id"]))
    return current


def test_captures_of_one_stream_share_nothing(capture):
    spaces = _Workspaces(7)
    eager = spaces.get(HOST, 5, 4096)
    held = []
    for capture["id"] in (1, 2):
        first = spaces.get(HOST, 5, 4096)
        assert first[0] != eager[0] and first[1] >= 4096
        held.append(spaces._captured[0, 5][1])
        assert spaces.get(HOST, 5, 4096) == first and spaces.get(HOST, 5, 64) == first
        assert not held[-1].any()
        other = spaces.get(HOST, 6, 4096)  # a stream that the capture forked to
        assert other[0] != first[0]
    assert held[0].data_ptr() != held[1].data_ptr()
    capture["id"] = 0
    assert spaces.get(HOST, 5, 4096) == eager


def test_a_larger_call_of_a_capture_gets_more(capture):
    spaces = _Workspaces(7, 16)
    capture["id"] = 3
    assert spaces.get(HOST, 5, 100)[1] >= 100
    got = spaces.get(HOST, 5, 1000)
    assert got[1] >= 1000 and not spaces._captured[0, 5][1][:16].any()
    assert spaces.get(HOST, 5, 0) == (0, 0)


def test_streams_keep_their_buffers(capture):
    spaces = _Workspaces(7)
    a, b = spaces.get(HOST, 1, 2000), spaces.get(HOST, 2, 2000)
    assert a[0] != b[0] and spaces.get(HOST, 1, 2000) == a
    assert spaces.get(HOST, 1, 3 << 20)[1] >= 3 << 20
