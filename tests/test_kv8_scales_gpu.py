"""Attention over blocks whose scales are zero, beside blocks of small values.

Tolerance, from the arithmetic: test_kv8_gpu.py's (weights of 11 bits, scores in
fp32, the result's own rounding), and what exponents of up to 128 cost, which are
rounded at 2^-18: five roundings, twice, of 0.7 2^-18 each are below 2^-14 of
sum p |v|.  No absolute term: small values count in full."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from light_vllm_b200 import _native, kv8_attention
from oracle import kv8 as okv8
from test_kv8_gpu import DEV, HALF, _codes, _layer, _np, _step, _tables

pytestmark = pytest.mark.gpu
BATCHES = {"tokens": [(500, 1), (47, 1), (3000, 1)], "drafts": [(500, 8), (100, 6)], "chunk": [(70, 150), (600, 40)]}


def _check(query, layer, step, tables, requests, code, scale):
    out = _np(kv8_attention(query, layer, step, scale=scale))
    keys = okv8.dequantise(_codes(layer.keys), _np(layer.key_scales), code)
    values = okv8.dequantise(_codes(layer.values), _np(layer.value_scales), code)
    want, size, reach = okv8.attend(_np(query), keys, values, tables, requests, scale)
    d = query.shape[-1]
    bound = size * (2.0 ** -11 + 2.0 ** -14 + 2 * (d + 16) * 2.0 ** -23 * reach[..., None]) + np.abs(want) * HALF[query.dtype]
    assert np.isfinite(out).all()
    worst = (np.abs(out - want) / np.maximum(bound, 1e-300)).max()
    assert worst <= 1.0, f"error is {worst:.2f} of its bound"
    assert _native.device_error() == 0


def _case(batch, heads, code, seed, size=1.0):
    requests = BATCHES[batch]
    tables, blocks = _tables(requests, 16, seed=seed)
    layer = _layer(blocks, heads[1], 16, heads[2], code, seed=seed)
    layer.value_scales.mul_(size)
    gen = torch.Generator(device=DEV).manual_seed(seed + 1)
    query = torch.randn((sum(n for _, n in requests), heads[0], heads[2]), device=DEV, generator=gen).to(torch.bfloat16)
    return query, layer, _step(tables, requests), tables, requests


@pytest.mark.parametrize("size", [2.0 ** -20, 2.0 ** -24, 2.0 ** -30, 2.0 ** -90])
@pytest.mark.parametrize("batch", BATCHES)
@pytest.mark.parametrize("heads,code", [((28, 4, 128), "int8"), ((14, 2, 64), "e4m3")])
def test_a_block_of_zeros_beside_small_values(size, batch, heads, code):
    """The zeros take their share of the weights and cost the others no bits."""

    query, layer, step, tables, requests = _case(batch, heads, code, 1, size)
    for t in tables:
        for b in (t[0], t[len(t) // 2]):
            layer.values[b] = 0
            layer.value_scales[b] = 0
    _check(query, layer, step, tables, requests, code, heads[2] ** -0.5)


@pytest.mark.parametrize("batch", BATCHES)
def test_nothing_but_zeros(batch):
    query, layer, step, tables, requests = _case(batch, (14, 2, 64), "int8", 2)
    layer.values.zero_()
    layer.value_scales.zero_()
    assert not kv8_attention(query, layer, step, scale=0.125).any()
    assert _native.device_error() == 0


def _as_if_zero(layer, blocks, side):
    """A side's scales at zero in some blocks, over whatever codes, and over codes of zero."""

    scales = getattr(layer, side + "_scales").clone()
    scales[blocks] = 0
    stale = layer._replace(**{side + "_scales": scales})
    codes = getattr(layer, side + "s").clone()
    codes.view(torch.uint8)[blocks] = 0
    return stale, stale._replace(**{side + "s": codes})


@pytest.mark.parametrize("batch", BATCHES)
@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_codes_under_a_key_scale_of_zero(batch, code):
    """A code stands for code * scale: under a scale that was set to zero it is a zero, bit for bit."""

    query, layer, step, tables, requests = _case(batch, (14, 2, 64), code, 3)
    stale, zeros = _as_if_zero(layer, sum((t[::2] for t in tables), []), "key")
    assert torch.equal(kv8_attention(query, stale, step, scale=0.125), kv8_attention(query, zeros, step, scale=0.125))
    _check(query, stale, step, tables, requests, code, 0.125)


@pytest.mark.parametrize("size", [1.0, 2.0 ** -40])
@pytest.mark.parametrize("batch", BATCHES)
@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_codes_under_a_value_scale_of_zero(batch, code, size):
    query, layer, step, tables, _ = _case(batch, (14, 2, 64), code, 4, size)
    stale, zeros = _as_if_zero(layer, sum((t[::2] for t in tables), []), "value")
    assert torch.equal(kv8_attention(query, stale, step, scale=0.125), kv8_attention(query, zeros, step, scale=0.125))
    assert _native.device_error() == 0
