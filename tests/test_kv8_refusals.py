"""What the 8-bit cache and the draft verification refuse, before any launch (CPU only)."""

from __future__ import annotations

import pytest
import torch

from light_vllm_b200 import KV8Layer, KV8Step, KVCacheError, _native, kv8_append, kv8_attention, kv8_read_blocks, verify_drafts


def _layer(dtype=torch.int8, shape=(4, 2, 16, 64), scales=(4, 2), scale_dtype=torch.float32):
    return KV8Layer(torch.zeros(shape, dtype=dtype), torch.zeros(shape, dtype=dtype), torch.zeros(scales, dtype=scale_dtype),
                    torch.zeros(scales, dtype=scale_dtype))


STEP = KV8Step(torch.zeros((1, 1), dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), 1, 1)
ROWS = torch.zeros((1, 2, 64), dtype=torch.float16)


@pytest.mark.parametrize("layer,message", [
    (_layer(torch.uint8), "int8 or float8_e4m3fn"),
    (_layer()._replace(values=torch.zeros((4, 2, 16, 64), dtype=torch.float8_e4m3fn)), "keys and values alike"),
    (_layer(shape=(4, 2, 16)), r"\[num_blocks, kv_heads, block_size, head_size\]"),
    (_layer()._replace(values=torch.zeros((4, 2, 32, 64), dtype=torch.int8)), r"\[num_blocks, kv_heads"),
    (_layer(scales=(4, 3)), "scales must be float32"),
    (_layer(scale_dtype=torch.float16), "scales must be float32"),
    (_layer()._replace(keys=torch.zeros((4, 2, 64, 16), dtype=torch.int8).transpose(2, 3)), "contiguous"),
    (_layer(), "one CUDA device"),
])
def test_layers(layer, message):
    for call in (lambda: kv8_attention(ROWS, layer, STEP, scale=1.0), lambda: kv8_append(None, ROWS, ROWS, layer, STEP),
                 lambda: kv8_read_blocks(layer, torch.zeros(1, dtype=torch.int32), dtype=torch.float16)):
        with pytest.raises(KVCacheError, match=message):
            call()


def _probs(rows=3, vocab=8):
    return torch.zeros((rows, vocab))


GOOD = dict(draft_tokens=torch.zeros(2, dtype=torch.int64), accept_uniform=torch.zeros(2), sample_uniform=torch.zeros(1),
            query_start=torch.zeros(2, dtype=torch.int32))


def test_verification_refuses_other_types_and_hosts():
    with pytest.raises(ValueError, match="float32"):
        verify_drafts(_probs().half(), **GOOD, max_query_len=3)
    with pytest.raises(ValueError, match="CUDA device"):
        verify_drafts(_probs(), **GOOD, max_query_len=3)


def _append(lib, **k):
    a = dict(hq=4, hkv=2, d=64, bs=16, dtype=0, code=0, n=1, tokens=1, key=16, key_stride=128, codes=16, positions=None,
             query=None, longest=1)
    a.update(k)
    return lib.lvb_kv8_append(a["query"], 256, a["query"], 256, a["key"], a["key_stride"], 16, 128, a["positions"], None, None, 0,
                              a["codes"], 16, 16, 16, 16, 1, 16, 16, a["n"], a["tokens"], a["longest"], a["hq"], a["hkv"],
                              a["d"], a["bs"], 4, a["dtype"], a["code"], None)


@pytest.mark.parametrize("change,status,message", [
    (dict(dtype=2), "INVALID", "unknown dtype"),
    (dict(code=2), "INVALID", "unknown code type"),
    (dict(n=-1), "INVALID", "batch size"),
    (dict(hkv=0), "INVALID", "KV head count"),
    (dict(d=80), "UNSUPPORTED", "head size 80"),
    (dict(bs=8), "UNSUPPORTED", "block size 8"),
    (dict(bs=24), "UNSUPPORTED", "block size 24"),
    (dict(hq=-1), "INVALID", "query head count"),
    (dict(key=None), "INVALID", "null pointer"),
    (dict(codes=8), "INVALID", "16-byte aligned"),
    (dict(key_stride=64), "INVALID", "strides must cover"),
    (dict(positions=16), "INVALID", "null pointer"),
    (dict(query=16), "INVALID", "null pointer"),
])
def test_append_entry(change, status, message):
    lib = _native.library()
    assert _append(lib, **change) == getattr(_native, f"LVB_ERR_{status}")
    assert message in lib.lvb_last_error().decode()


def test_append_of_nothing_launches_nothing():
    assert _append(_native.library(), tokens=0) == _native.LVB_OK
    assert _append(_native.library(), n=0) == _native.LVB_OK


def _attention(lib, **k):
    a = dict(hq=4, hkv=2, d=64, bs=16, dtype=0, code=0, n=1, tokens=1, longest=1, max_seq=16, query=16, out=16, q_stride=256)
    a.update(k)
    return lib.lvb_kv8_attention(a["query"], a["q_stride"], 16, 16, 16, 16, a["out"], 256, 16, 1, 16, 16, a["n"], a["tokens"],
                                 a["longest"], a["max_seq"], a["hq"], a["hkv"], a["d"], a["bs"], 4, 1.0, a["dtype"], a["code"],
                                 None, 0, None)


@pytest.mark.parametrize("change,status,message", [
    (dict(dtype=-1), "INVALID", "unknown dtype"),
    (dict(hq=3), "INVALID", "3 query heads over 2 KV heads"),
    (dict(hq=0), "INVALID", "query heads"),
    (dict(d=256), "UNSUPPORTED", "head size 256"),
    (dict(bs=0), "UNSUPPORTED", "block size 0"),
    (dict(max_seq=-1), "INVALID", "longest sequence"),
    (dict(query=None), "INVALID", "null pointer"),
    (dict(out=None), "INVALID", "null pointer"),
    (dict(q_stride=128), "INVALID", "strides must cover"),
])
def test_attention_entry(change, status, message):
    lib = _native.library()
    assert _attention(lib, **change) == getattr(_native, f"LVB_ERR_{status}")
    assert message in lib.lvb_last_error().decode()


def test_read_and_verify_entries():
    lib = _native.library()
    read = lambda ids, out, d=64: lib.lvb_kv8_read_blocks(16, 16, 16, 16, ids, 1, out, 16, 2, d, 16, 4, 0, 0, None)  # noqa: E731
    assert read(None, 16) == _native.LVB_ERR_INVALID and b"null pointer" in lib.lvb_last_error()
    assert read(16, 8) == _native.LVB_ERR_INVALID and b"16-byte aligned" in lib.lvb_last_error()
    assert read(16, 16, 96) == _native.LVB_ERR_UNSUPPORTED

    def verify(n=1, rows=1, vocab=8, stride=8, target=16, drafts=None):
        return lib.lvb_verify_drafts(target, stride, None, 0, drafts, drafts, 16, 16, 16, 16, n, rows, 2, vocab, None, 0, None)

    for change, message in ((dict(vocab=0), b"vocabulary size"), (dict(stride=7), b"strides"), (dict(target=None), b"null pointer"),
                            (dict(rows=2), b"null pointer"), (dict(rows=0), b"every request needs a row"), (dict(n=-1), b"batch")):
        assert verify(**change) == _native.LVB_ERR_INVALID
        assert message in lib.lvb_last_error()
    assert verify(n=0) == _native.LVB_OK


def test_verification_of_more_words_than_its_sums_hold():
    lib = _native.library()
    words = (1 << 22) + 1
    assert lib.lvb_verify_drafts(16, words, None, 0, None, None, 16, 16, 16, 16, 1, 1, 2, words, None, 0, None) == _native.LVB_ERR_UNSUPPORTED
    assert b"2^22" in lib.lvb_last_error()
