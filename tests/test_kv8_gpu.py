"""The 8-bit paged cache on the GPU against its formulas in 64 bits.

Tolerances, from the arithmetic (u = 2^-24 is half a unit in the last place of
fp32, h = 2^-11 or 2^-8 that of fp16 or bf16):

* a rotated value carries at most 2 u (|x1 c| + |x2 s|), and the largest of a
  pair is at least 1 / sqrt(2) of the pair's norm, so a block's scale is within
  16 u of its exact value, division and product included;
* a code is the nearest one for a value within that error: half a step, plus
  M * 16 u of a step (int8: 127 * 16 u < 2e-4; e4m3 is relative: 2e-5);
* attention: the weights enter the second product in 16 bits (2^-11 each, of
  sum p |v|), a score's fp32 sum of D products, truncated or rounded, is within
  (D + 16) 2^-23 of scale * sum |q k|, which a weight carries twice (itself and
  through the sum), and the result is rounded to the query's type (h).
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from light_vllm_b200 import KV8Layer, KV8Step, _native, kv8_append, kv8_attention, kv8_read_blocks
from oracle import kv8 as okv8

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
U = 2.0 ** -24
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _np(t):
    return t.detach().float().cpu().numpy()


def _codes(t):
    """Codes as the oracle takes them."""

    return t.cpu().numpy() if t.dtype == torch.int8 else t.view(torch.uint8).cpu().numpy()


def _step(tables, requests, *, max_query=None, max_seq=None):
    starts = np.cumsum([0] + [n for _, n in requests])
    width = max(1, max((len(t) for t in tables), default=1))
    rows = [list(t) + [0] * (width - len(t)) for t in tables]
    return KV8Step(torch.tensor(rows, dtype=torch.int32, device=DEV).view(len(tables), width),
                   torch.tensor([c for c, _ in requests], dtype=torch.int32, device=DEV),
                   torch.tensor(starts, dtype=torch.int32, device=DEV),
                   max([n for _, n in requests] + [0]) if max_query is None else max_query,
                   max([c + n for c, n in requests] + [0]) if max_seq is None else max_seq)


def _tables(requests, bs, spare=3, seed=0):
    """Blocks of each request from a permuted pool; returns (tables, pool size)."""

    need = [-(-(c + n) // bs) for c, n in requests]
    ids = np.random.default_rng(seed).permutation(sum(need) + spare).tolist()
    tables, at = [], 0
    for k in need:
        tables.append(ids[at:at + k])
        at += k
    return tables, sum(need) + spare


def _layer(blocks, hkv, bs, d, code, seed=0, size=1.0):
    """Random codes and scales, as earlier steps leave them (no NaN patterns)."""

    gen = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn((2, blocks, hkv, bs, d), device=DEV, generator=gen)
    x[..., 5::31] *= 4
    scales = x.abs().amax(dim=(3, 4)) / okv8.TOP[code]
    y = x / scales[..., None, None]
    codes = (y.round() if code == "int8" else y).to(CODES[code])
    scales = scales * size
    return KV8Layer(codes[0].contiguous(), codes[1].contiguous(), scales[0].contiguous(), scales[1].contiguous())


def _check_attention(query, layer, step, tables, requests, code, scale, out):
    keys = okv8.dequantise(_codes(layer.keys), _np(layer.key_scales), code)
    values = okv8.dequantise(_codes(layer.values), _np(layer.value_scales), code)
    # slots that no request has reached may hold anything
    want, size, reach = okv8.attend(_np(query), np.nan_to_num(keys), np.nan_to_num(values), tables, requests, scale)
    d = query.shape[-1]
    bound = size * (2.0 ** -11 + 2 * (d + 16) * 2.0 ** -23 * reach[..., None]) + np.abs(want) * HALF[query.dtype] + 1e-7
    got = _np(out)
    assert np.isfinite(got).all()
    worst = (np.abs(got - want) / bound).max() if got.size else 0.0
    assert worst <= 1.0, f"error is {worst:.2f} of its bound"
    assert _native.device_error() == 0


BATCHES = [
    [(0, 1)],
    [(14, 1), (15, 1), (16, 1), (17, 1)],
    [(31, 1), (0, 0), (33, 1), (7, 0)],
    [(100, 5), (0, 3), (47, 1), (63, 2)],
    [(37, 40), (0, 131), (250, 1)],
    [(0, 257), (600, 129)],
    [(3000, 1), (5, 1), (777, 4)],
]
HEADS = [(4, 4, 64), (14, 2, 64), (28, 4, 128), (16, 1, 128), (40, 1, 64)]


@pytest.mark.parametrize("requests", BATCHES, ids=lambda b: "+".join(f"{c}.{n}" for c, n in b))
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("code,dtype,bs", [("int8", torch.float16, 16), ("e4m3", torch.bfloat16, 32),
                                           ("int8", torch.bfloat16, 48), ("e4m3", torch.float16, 16)])
def test_attention(requests, heads, code, dtype, bs):
    hq, hkv, d = heads
    tables, blocks = _tables(requests, bs)
    layer = _layer(blocks, hkv, bs, d, code, seed=1)
    tokens = sum(n for _, n in requests)
    gen = torch.Generator(device=DEV).manual_seed(2)
    query = (torch.randn((tokens, hq, d), device=DEV, generator=gen) * 2).to(dtype)
    step = _step(tables, requests)
    out = kv8_attention(query, layer, step, scale=d ** -0.5)
    _check_attention(query, layer, step, tables, requests, code, d ** -0.5, out)
    again = kv8_attention(query, layer, step, scale=d ** -0.5)
    assert torch.equal(out, again)


@pytest.mark.parametrize("requests", [[(5, 1), (200, 1)], [(5, 3), (300, 200)]], ids=["tokens", "chunks"])
@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_attention_ignores_what_lies_past_the_end(requests, code):
    """NaN patterns, infinite scales and NaN scales in slots and blocks that no query reaches."""

    hq, hkv, d, bs = 14, 2, 128, 16
    tables, blocks = _tables(requests, bs)
    layer = _layer(blocks, hkv, bs, d, code, seed=3)
    used = {b for t in tables for b in t}
    for r, (c, n) in enumerate(requests):
        last = (c + n) % bs
        if last:
            for t in (layer.keys, layer.values):
                t.view(torch.uint8)[tables[r][-1], :, last:] = 0x7F
    for b in set(range(blocks)) - used:
        layer.keys.view(torch.uint8)[b] = 0xFF
        layer.key_scales[b] = float("nan")
        layer.value_scales[b] = float("inf")
    query = torch.randn((sum(n for _, n in requests), hq, d), device=DEV, dtype=torch.float16)
    step = _step(tables, requests)
    out = kv8_attention(query, layer, step, scale=0.1)
    _check_attention(query, layer, step, tables, requests, code, 0.1, out)


@pytest.mark.parametrize("size", [1e-6, 3e3])
@pytest.mark.parametrize("requests", [[(500, 1), (3, 1)], [(70, 150)]], ids=["tokens", "chunk"])
def test_attention_with_blocks_of_very_different_size(size, requests):
    """Neighbouring blocks whose scales differ by many powers of two, and blocks of zeros."""

    hq, hkv, d, bs = 28, 4, 128, 16
    tables, blocks = _tables(requests, bs)
    layer = _layer(blocks, hkv, bs, d, "int8", seed=4)
    layer.value_scales[::3] *= size
    layer.key_scales[::4] *= 0.01
    zero = tables[0][1 % len(tables[0])]
    layer.values[zero] = 0
    layer.value_scales[zero] = 0
    layer.keys[zero] = 0
    layer.key_scales[zero] = 0
    query = torch.randn((sum(n for _, n in requests), hq, d), device=DEV).to(torch.bfloat16)
    step = _step(tables, requests)
    out = kv8_attention(query, layer, step, scale=d ** -0.5)
    _check_attention(query, layer, step, tables, requests, "int8", d ** -0.5, out)


@pytest.mark.parametrize("magnitude", [1e-30, 1e-6, 3e4, 1e30])
def test_attention_of_queries_of_any_size(magnitude):
    """bf16 queries reach far past fp16's range; the scale brings the scores back."""

    requests, bs, d = [(90, 1), (10, 30)], 16, 64
    tables, blocks = _tables(requests, bs)
    layer = _layer(blocks, 2, bs, d, "e4m3", seed=5)
    query = (torch.randn((31, 8, d), device=DEV) * magnitude).to(torch.bfloat16)
    step = _step(tables, requests)
    scale = 0.1 / magnitude
    out = kv8_attention(query, layer, step, scale=scale)
    _check_attention(query, layer, step, tables, requests, "e4m3", scale, out)


def test_attention_of_strided_rows_and_a_given_output():
    requests, bs, d = [(33, 1), (20, 3)], 16, 64
    tables, blocks = _tables(requests, bs)
    layer = _layer(blocks, 2, bs, d, "int8", seed=6)
    step = _step(tables, requests)
    merged = torch.randn((4, 18, d), device=DEV).half()
    query = merged[:, :14]
    odd = torch.randn(4 * 14 * d + 1, device=DEV).half()[1:].view(4, 14, d)  # 2-byte aligned
    turned = query.transpose(0, 1).contiguous().transpose(0, 1)  # heads outermost
    wide = torch.zeros((4, 20, d), device=DEV, dtype=torch.float16)
    want = kv8_attention(query.contiguous(), layer, step, scale=0.2)
    assert torch.equal(kv8_attention(query, layer, step, scale=0.2, out=wide[:, 2:16]), want)
    assert torch.equal(wide[:, 2:16], want) and not wide[:, :2].any() and not wide[:, 16:].any()
    assert torch.equal(kv8_attention(turned, layer, step, scale=0.2), want)
    odd.copy_(query)
    assert torch.equal(kv8_attention(odd, layer, step, scale=0.2), want)


def test_attention_does_not_depend_on_the_longest_sequence_named():
    """max_seq_len guides the split; results stay within the tolerance whatever it says."""

    requests, bs, d = [(2000, 1), (1200, 2)], 16, 128
    tables, blocks = _tables(requests, bs)
    layer = _layer(blocks, 4, bs, d, "int8", seed=7)
    query = torch.randn((3, 28, d), device=DEV).half()
    for named in (0, 16, 100000):
        step = _step(tables, requests, max_seq=named)
        out = kv8_attention(query, layer, step, scale=d ** -0.5)
        _check_attention(query, layer, step, tables, requests, "int8", d ** -0.5, out)


def test_caches_past_4_gib():
    """Block offsets that do not fit 32 bits."""

    bs, d, blocks = 16, 128, 2_200_000
    layer = KV8Layer(*(torch.zeros((blocks, 1, bs, d), dtype=torch.int8, device=DEV) for _ in range(2)),
                     *(torch.zeros((blocks, 1), device=DEV) for _ in range(2)))
    tables, requests = [[blocks - 1, 3, blocks - 70000]], [(35, 1)]
    small = _layer(blocks=3, hkv=1, bs=bs, d=d, code="int8", seed=8)
    for i, b in enumerate(tables[0]):
        for big, part in zip(layer, small):
            big[b] = part[i]
    gen = torch.Generator(device=DEV).manual_seed(9)
    query, key, value = (torch.randn((1, h, d), device=DEV, generator=gen).half() for h in (4, 1, 1))
    step = _step(tables, requests)
    near = _step([[0, 1, 2]], requests)
    kv8_append(None, key, value, layer, step)
    kv8_append(None, key, value, small, near)
    for i, b in enumerate(tables[0]):
        for big, part in zip(layer, small):
            assert torch.equal(big[b], part[i])
    ids = torch.tensor(tables[0], dtype=torch.int32, device=DEV)
    for got, want in zip(kv8_read_blocks(layer, ids, dtype=torch.float16),
                         kv8_read_blocks(small, torch.arange(3, dtype=torch.int32, device=DEV), dtype=torch.float16)):
        assert torch.equal(got, want)
    assert torch.equal(kv8_attention(query, layer, step, scale=0.1), kv8_attention(query, small, near, scale=0.1))
    long_query = torch.randn((36, 20, d), device=DEV, generator=gen).half()
    far, close = _step(tables, [(0, 36)]), _step([[0, 1, 2]], [(0, 36)])
    assert torch.equal(kv8_attention(long_query, layer, far, scale=0.1), kv8_attention(long_query, small, close, scale=0.1))


# ------------------------------------------------------------------- append
def _rows(tokens, hq, hkv, d, dtype, seed, size=1.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    qkv = (torch.randn((tokens, (hq + 2 * hkv) * d), device=DEV, generator=gen) * size).to(dtype)
    return qkv.view(tokens, hq + 2 * hkv, d).split((hq, hkv, hkv), dim=1)


def _rope(rows, d, dtype):
    angle = torch.outer(torch.arange(rows, device=DEV, dtype=torch.float32),
                        1e4 ** (-torch.arange(0, d, 2, device=DEV, dtype=torch.float32) / d)).repeat(1, 2)
    return angle.cos().to(dtype), angle.sin().to(dtype)


def _check_append(before, after, rows, tables, requests, code, bs):
    """rows: per side the exact new rows [tokens, heads, d] in 64 bits."""

    slack = 2e-4 if code == "int8" else 2e-5
    for side, new in rows.items():
        i = 0 if side == "key" else 1
        old_codes, codes = _codes(before[i]), _codes(after[i])
        old_scales, scales = _np(before[i + 2]).astype(np.float64), _np(after[i + 2]).astype(np.float64)
        touched, t0 = set(), 0
        for r, (c, n) in enumerate(requests):
            for b in range(c // bs, -(-(c + n) // bs)) if n else ():
                phys = tables[r][b]
                touched.add(phys)
                lo, hi = max(c, b * bs) - b * bs, min(c + n, (b + 1) * bs) - b * bs
                x = new[t0 + b * bs + lo - c: t0 + b * bs + hi - c].transpose(1, 0, 2)  # [heads, new, d]
                top = np.abs(x).max(axis=(1, 2)) / okv8.TOP[code]
                s0 = old_scales[phys] if lo else np.zeros_like(top)
                want = np.maximum(s0, top)
                assert (np.abs(scales[phys] - want) <= 16 * U * want).all()
                s1 = scales[phys][:, None, None]
                got = okv8.code_values(codes[phys], code)
                held = okv8.code_values(old_codes[phys], code)
                safe = np.where(s1 > 0, s1, 1)
                y = x / safe
                assert (np.abs(got[:, lo:hi] - y) <= okv8.half_step(y, code) * (1 + slack) + slack).all()
                y = held[:, :lo] * (s0[:, None, None] / safe)
                assert (np.abs(got[:, :lo] - y) <= okv8.half_step(y, code) * (1 + slack) + slack).all()
                same = scales[phys] == old_scales[phys]
                assert (codes[phys][same, :lo] == old_codes[phys][same, :lo]).all()
                assert (codes[phys][:, hi:] == old_codes[phys][:, hi:]).all()
            t0 += n
        others = [b for b in range(codes.shape[0]) if b not in touched]
        assert (codes[others] == old_codes[others]).all() and (scales[others] == old_scales[others]).all()
    assert _native.device_error() == 0


APPENDS = BATCHES + [[(16, 16)], [(8, 24), (0, 16), (15, 2)], [(1, 1)] * 40]


@pytest.mark.parametrize("requests", APPENDS, ids=lambda b: f"{b[0]}x{len(b)}")
@pytest.mark.parametrize("heads", [(4, 4, 64), (28, 4, 128), (7, 1, 64)], ids=str)
@pytest.mark.parametrize("code,dtype,bs", [("int8", torch.float16, 16), ("e4m3", torch.bfloat16, 16),
                                           ("int8", torch.bfloat16, 64), ("e4m3", torch.float16, 48)])
def test_append(requests, heads, code, dtype, bs):
    hq, hkv, d = heads
    tables, blocks = _tables(requests, bs)
    layer = _layer(blocks, hkv, bs, d, code, seed=11, size=0.7)
    before = [t.clone() for t in layer]
    tokens = sum(n for _, n in requests)
    query, key, value = _rows(tokens, hq, hkv, d, dtype, seed=12)
    kept = query.clone()
    cos, sin = _rope(4000, d, dtype)
    at = [c + i for c, n in requests for i in range(n)]
    positions = torch.tensor(at, dtype=torch.int32, device=DEV)
    step = _step(tables, requests)
    out = kv8_append(query, key, value, layer, step, positions=positions, cos=cos, sin=sin)
    c, s = _np(cos)[at], _np(sin)[at]
    exact = okv8.rotate(_np(query), c, s)
    norm = np.abs(_np(query)).max() if tokens else 0
    assert (np.abs(_np(out) - exact) <= np.abs(exact) * HALF[dtype] * (1 + 1e-3) + 4 * U * norm + 2.0 ** -25).all()
    assert torch.equal(query, kept)
    _check_append(before, layer, {"key": okv8.rotate(_np(key), c, s), "value": _np(value).astype(np.float64)}, tables,
                  requests, code, bs)
    # the same rows again leave the cache as it is, and rotate in place alike
    after = [t.clone() for t in layer]
    assert kv8_append(query, key, value, layer, step, positions=positions, cos=cos, sin=sin, query_out=query) is query
    assert torch.equal(query, out)
    for x, y in zip(after, layer):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_append_token_by_token_keeps_earlier_values(code):
    """A block filled one token at a time: growing scales round earlier codes anew, and every
    rounding is at most half a step of the scale it was made with."""

    hkv, d, bs = 2, 64, 16
    layer = KV8Layer(*(torch.zeros((2, hkv, bs, d), dtype=torch.int8, device=DEV).view(CODES[code]) for _ in range(2)),
                     *(torch.full((2, hkv), 9.0, device=DEV) for _ in range(2)))  # stale scales of an earlier owner
    gen = torch.Generator(device=DEV).manual_seed(13)
    grow = torch.linspace(0.2, 3, 20, device=DEV)[:, None, None]
    key, value = ((torch.randn((20, hkv, d), device=DEV, generator=gen) * grow).half() for _ in range(2))
    for p in range(20):
        kv8_append(None, key[p:p + 1], value[p:p + 1], layer, _step([[1, 0]], [(p, 1)]))
    ids = torch.tensor([1, 0], dtype=torch.int32, device=DEV)
    for got, x, scales in zip(kv8_read_blocks(layer, ids, dtype=torch.float16), (key, value), layer[2:]):
        got = got.transpose(0, 1).reshape(hkv, -1, d)[:, :20].transpose(0, 1)
        for blk, (lo, hi) in zip((1, 0), ((0, 16), (16, 20))):
            s = _np(scales)[blk][None, :, None]
            top = np.abs(_np(x[lo:hi])).max(axis=(0, 2)) / okv8.TOP[code]
            assert np.allclose(s[0, :, 0], top, rtol=1e-6)
            steps = okv8.half_step(np.abs(_np(x[lo:hi])) / s, code) * s
            # at most hi - lo roundings, with scales no larger than the last
            assert (np.abs(_np(got[lo:hi]) - _np(x[lo:hi])) <= steps * (hi - lo) * 1.1 + 1e-3).all()
            # and on the whole far fewer
            assert np.abs(_np(got[lo:hi]) - _np(x[lo:hi])).mean() <= 1.5 * steps.mean()


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_append_of_zeros_tiny_values_and_what_is_not_finite(code):
    hkv, d, bs = 1, 64, 16
    top = okv8.TOP[code]
    for rows, want in (([0.0, -0.0], [0, 0]), ([1e-35, -1e-33], [0, 0]), ([float("nan"), 2.0], [0, top]),
                       ([float("inf"), 1.0], [top, 0]), ([-float("inf"), 1e30], [-top, 0])):
        layer = _layer(2, hkv, bs, d, code, seed=14)
        x = torch.tensor(rows, device=DEV).view(2, 1, 1).expand(2, hkv, d).to(torch.bfloat16).contiguous()
        kv8_append(None, x, x, layer, _step([[1]], [(0, 2)]))
        for codes, scales in ((layer.keys, layer.key_scales), (layer.values, layer.value_scales)):
            got = okv8.code_values(_codes(codes[1:]), code)[0, :, :2, 0]
            assert got.tolist() == [[float(w) for w in want]]
            assert np.isfinite(_np(scales)[1]).all()
            assert (want != [0, 0]) or _np(scales)[1].tolist() == [0.0]
    assert _native.device_error() == 0


@pytest.mark.parametrize("bs", [16, 64])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_read_blocks(code, dtype, bs):
    layer = _layer(7, 3, bs, 64, code, seed=15)
    ids = torch.tensor([6, 0, 0, 3], dtype=torch.int32, device=DEV)
    for got, codes, scales in zip(kv8_read_blocks(layer, ids, dtype=dtype), layer[:2], layer[2:]):
        want = torch.from_numpy(okv8.code_values(_codes(codes), code)[ids.cpu().numpy()]).to(DEV).float()
        assert torch.equal(got, (want * scales[ids.long()][..., None, None]).to(dtype))
    empty = kv8_read_blocks(layer, ids[:0], dtype=dtype)
    assert empty[0].shape == (0, 3, bs, 64)


def test_out_of_range_metadata_is_reported_and_left_out():
    """Block ids, positions and query starts that only the device sees."""

    hq, hkv, d, bs = 4, 2, 64, 16
    layer = _layer(4, hkv, bs, d, "int8", seed=16)
    before = [t.clone() for t in layer]
    query, key, value = _rows(2, hq, hkv, d, torch.float16, seed=17)
    cos, sin = _rope(32, d, torch.float16)

    def step(tables, computed, start, longest=1):
        return KV8Step(torch.tensor(tables, dtype=torch.int32, device=DEV), torch.tensor(computed, dtype=torch.int32, device=DEV),
                       torch.tensor(start, dtype=torch.int32, device=DEV), longest, 32)

    ok = torch.tensor([3, 4], dtype=torch.int32, device=DEV)
    bad = {
        "block id": step([[4], [-1]], [3, 4], [0, 1, 2]),
        "past the table": step([[1], [2]], [16, 40], [0, 1, 2]),
        "past the batch": step([[1], [2]], [3, 4], [0, 3, 5], 3),
        "longer than named": step([[1]], [3], [0, 2], 1),
        "negative": step([[1], [2]], [-1, -40], [0, 1, 2]),
    }
    for name, s in bad.items():
        kv8_append(query, key, value, layer, s, positions=ok, cos=cos, sin=sin)
        assert _native.device_error() == 2, name
        kv8_attention(query, layer, s, scale=0.1)
        assert _native.device_error() == 2, name
    kv8_append(query, key, value, layer, step([[1], [2]], [3, 4], [0, 1, 2]),
               positions=torch.tensor([32, -1], dtype=torch.int32, device=DEV), cos=cos, sin=sin)
    assert _native.device_error() == 2
    # a token whose position is outside the tables leaves its key out; its value needs no rotation
    for x, y in zip((layer.keys, layer.key_scales), (before[0], before[2])):
        assert torch.equal(x, y)
    got = kv8_read_blocks(layer, torch.tensor([9, 1], dtype=torch.int32, device=DEV), dtype=torch.float16)
    assert _native.device_error() == 2 and not got[0][0].any() and got[0][1].any()


@pytest.mark.parametrize("heads,query", [((14, 2, 64), 8), ((14, 2, 64), 9), ((16, 1, 64), 3), ((64, 1, 64), 1), ((16, 1, 128), 4),
                                         ((28, 4, 128), 6), ((64, 1, 128), 1), ((24, 8, 64), 13), ((33, 1, 64), 1)], ids=str)
@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_attention_of_rows_in_two_groups(heads, query, code):
    """33 to 64 query rows of a KV head: one or two groups of the decode kernel's."""

    requests = [(700, query), (0, query), (15, 1), (2040, max(1, query - 1)), (64, 0), (333, query)]
    hq, hkv, d = heads
    tables, blocks = _tables(requests, 16, seed=3)
    layer = _layer(blocks, hkv, 16, d, code, seed=4)
    step = _step(tables, requests)
    gen = torch.Generator(device=DEV).manual_seed(5)
    query_rows = torch.randn((sum(n for _, n in requests), hq, d), device=DEV, generator=gen).to(torch.bfloat16)
    out = kv8_attention(query_rows, layer, step, scale=d ** -0.5)
    _check_attention(query_rows, layer, step, tables, requests, code, d ** -0.5, out)
