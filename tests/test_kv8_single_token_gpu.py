"""Rows of one token out of [heads, tokens, head_size] storage: their token stride
means nothing."""

from __future__ import annotations

import pytest
import torch

from light_vllm_b200 import _native, kv8_append, kv8_attention
from test_kv8_gpu import DEV, _layer, _rope, _step

pytestmark = pytest.mark.gpu


def _turned(x):
    """The same values [1, heads, d] with heads outermost in memory: token stride d."""

    y = x.transpose(0, 1).clone(memory_format=torch.contiguous_format).transpose(0, 1)
    assert y.stride(0) == x.shape[2] and torch.equal(x, y)
    return y


def _rows(heads, d, dtype):
    gen = torch.Generator(device=DEV).manual_seed(1)
    return [torch.randn((1, h, d), device=DEV, generator=gen).to(dtype) for h in heads]


@pytest.mark.parametrize("heads", [(8, 2, 64), (28, 4, 128), (64, 1, 128)], ids=str)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rotated", [False, True])
def test_one_token_with_heads_outermost(heads, dtype, rotated):
    hq, hkv, d = heads
    layers = [_layer(4, hkv, 16, d, "int8", seed=2) for _ in range(2)]
    step = _step([[2, 0, 1]], [(36, 1)])
    query, key, value = _rows((hq, hkv, hkv), d, dtype)
    turn = {}
    if rotated:
        cos, sin = _rope(64, d, dtype)
        turn = dict(positions=torch.tensor([36], dtype=torch.int32, device=DEV), cos=cos, sin=sin)
    got, want = (kv8_append(f(query) if rotated else None, f(key), f(value), layer, step, **turn)
                 for f, layer in zip((_turned, lambda x: x), layers))
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(*layers))
    if rotated:
        assert torch.equal(got, want)
        given = _turned(torch.zeros_like(query))
        assert kv8_append(query, key, value, layers[0], step, query_out=given, **turn) is given and torch.equal(given, want)
    want = kv8_attention(query, layers[0], step, scale=0.125)
    given = _turned(torch.zeros_like(query))
    assert torch.equal(kv8_attention(_turned(query), layers[0], step, scale=0.125), want)
    assert kv8_attention(_turned(query), layers[0], step, scale=0.125, out=given) is given and torch.equal(given, want)
    assert _native.device_error() == 0


def test_one_token_of_a_stride_that_is_no_multiple_of_16_bytes():
    layer = _layer(2, 2, 16, 64, "e4m3", seed=3)
    step = _step([[1]], [(9, 1)])
    query, = _rows((8,), 64, torch.float16)
    odd = query.as_strided(query.shape, (513, 64, 1))
    out = torch.zeros_like(query).as_strided(query.shape, (3, 64, 1))
    want = kv8_attention(query, layer, step, scale=0.125)
    assert torch.equal(kv8_attention(odd, layer, step, scale=0.125, out=out), want)
    assert torch.equal(out, want)


def test_one_kv_head_of_any_head_stride():
    """A head stride means nothing where there is one head."""

    layers = [_layer(3, 1, 16, 64, "int8", seed=4) for _ in range(2)]
    step = _step([[2, 1]], [(14, 3)])
    key, value = (torch.randn((3, 1, 64), device=DEV).half() for _ in range(2))
    kv8_append(None, key, value, layers[0], step)
    kv8_append(None, key.as_strided(key.shape, (64, 7, 1)), value.as_strided(value.shape, (64, 1, 1)), layers[1], step)
    assert all(torch.equal(a, b) for a, b in zip(*layers))
