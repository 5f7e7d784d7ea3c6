"""The C entry points that take a block table's columns and row stride apart (CPU only)."""

from __future__ import annotations

import pytest

from light_vllm_b200 import _native


def _append(lib, cols, stride):
    return lib.lvb_kv8_append_strided(None, 0, None, 0, 16, 128, 16, 128, None, None, None, 0, 16, 16, 16, 16, 16, cols, stride,
                                      16, 16, 1, 0, 1, 4, 2, 64, 16, 4, 0, 0, None)


def _attention(lib, cols, stride):
    return lib.lvb_kv8_attention_strided(16, 256, 16, 16, 16, 16, 16, 256, 16, cols, stride, 16, 16, 1, 0, 1, 16, 4, 2, 64, 16,
                                         4, 1.0, 0, 0, None, 0, None)


@pytest.mark.parametrize("call", [_append, _attention])
def test_columns_and_stride(call):
    lib = _native.library()
    for cols, stride in ((-1, 4), (4, -1), (1 << 31, 4), (4, 1 << 31)):
        assert call(lib, cols, stride) == _native.LVB_ERR_INVALID
        assert b"invalid batch size" in lib.lvb_last_error()
    for cols, stride in ((4, 0), (4, 1), (4, 9), (0, 0)):  # no tokens: nothing is launched
        assert call(lib, cols, stride) == _native.LVB_OK
