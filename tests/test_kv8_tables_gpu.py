"""Block tables whose rows do not lie one after the other: columns of a wider
buffer, one row for every request, a column turned into a row.  A table is as
long as it has columns, whatever its stride."""

from __future__ import annotations

import pytest
import torch

from light_vllm_b200 import KV8Step, _native, kv8_append, kv8_attention
from test_kv8_gpu import DEV, _layer, _rows, _step, _tables

pytestmark = pytest.mark.gpu
HEADS = (14, 2, 64)
# Single tokens, drafts in two row groups, prompt chunks beside tokens.
BATCHES = {"tokens": [(40, 1), (15, 1), (100, 1)], "drafts": [(60, 8), (3, 8), (90, 5)], "chunks": [(20, 70), (90, 1), (0, 120)]}


def _bits(layer):
    return [t.view(torch.uint8).clone() for t in layer]


def _new(requests, code="int8"):
    tables, blocks = _tables(requests, 16, spare=8)
    used = {b for t in tables for b in t}
    layer = _layer(blocks, HEADS[1], 16, HEADS[2], code, seed=1)
    return tables, layer, _step(tables, requests), [b for b in range(blocks) if b not in used]


def _run(layer, step, rows):
    query, key, value = rows
    kv8_append(None, key, value, layer, step)
    out = torch.full_like(query, 7.0)
    kv8_attention(query, layer, step, scale=0.125, out=out)
    return out


@pytest.mark.parametrize("batch", BATCHES)
def test_columns_of_a_wider_buffer(batch):
    requests = BATCHES[batch]
    _, layer, step, spare = _new(requests)
    _, other, _, _ = _new(requests)
    n, width = step.block_tables.shape
    wide = torch.full((n, width + 5), spare[0], dtype=torch.int32, device=DEV)
    wide[:, 3:3 + width] = step.block_tables
    rows = _rows(sum(q for _, q in requests), *HEADS, torch.float16, seed=2)
    want = _run(layer, step, rows)
    got = _run(other, step._replace(block_tables=wide[:, 3:3 + width]), rows)
    assert torch.equal(got, want)
    assert all(torch.equal(a, b) for a, b in zip(_bits(layer), _bits(other)))
    assert _native.device_error() == 0


@pytest.mark.parametrize("batch", BATCHES)
@pytest.mark.parametrize("late", [0, 2])
def test_a_context_past_the_columns_is_reported_and_left_out(batch, late):
    """The columns beyond the table name blocks of nobody: they must stay as they are, and so must the
    request's output rows, while the other requests run as ever."""

    requests = BATCHES[batch]
    tables, layer, step, spare = _new(requests)
    _, other, _, _ = _new(requests)
    n, width = step.block_tables.shape
    # the columns follow the table directly; the last row ends with its buffer
    wide = torch.full((n, width + 4), spare[1], dtype=torch.int32, device=DEV)
    wide[:, :width] = step.block_tables
    rows = _rows(sum(q for _, q in requests), *HEADS, torch.float16, seed=3)
    want = _run(layer, step, rows)
    assert _native.device_error() == 0
    computed = step.num_computed.clone()
    computed[late] = 16 * width - requests[late][1] + 1  # one token more than the columns hold
    before = _bits(other)
    got = _run(other, step._replace(block_tables=wide[:, :width], num_computed=computed), rows)
    assert _native.device_error() == 2
    after = _bits(other)
    mine = set(tables[late])
    for old, new, done in zip(before, after, _bits(layer)):
        for b in range(old.shape[0]):
            assert torch.equal(new[b], old[b] if b in mine else done[b])
    at = 0
    for r, (_, q) in enumerate(requests):
        if r == late:
            assert (got[at:at + q] == 7.0).all()
        else:
            assert torch.equal(got[at:at + q], want[at:at + q])
        at += q


@pytest.mark.parametrize("requests", [[(40, 1), (45, 1), (17, 1)], [(30, 18), (0, 48), (11, 9)]], ids=["tokens", "chunks"])
def test_one_row_for_every_request(requests):
    """Requests that read the same blocks."""

    layer = _layer(5, HEADS[1], 16, HEADS[2], "e4m3", seed=4)
    row = torch.tensor([[4, 1, 2]], dtype=torch.int32, device=DEV)
    step = _step([[4, 1, 2]] * len(requests), requests)
    query = _rows(sum(q for _, q in requests), *HEADS, torch.bfloat16, seed=5)[0]
    want = kv8_attention(query, layer, step, scale=0.125)
    shared = step._replace(block_tables=row.expand(len(requests), -1))
    assert shared.block_tables.stride(0) == 0
    assert torch.equal(kv8_attention(query, layer, shared, scale=0.125), want)
    assert _native.device_error() == 0


def test_a_column_turned_into_a_row():
    layer, other = (_layer(5, HEADS[1], 16, HEADS[2], "int8", seed=6) for _ in range(2))
    column = torch.tensor([[4], [1], [2]], dtype=torch.int32, device=DEV)
    step = _step([[4, 1, 2]], [(40, 1)])
    turned = KV8Step(column.t(), *step[1:])
    assert turned.block_tables.stride() == (1, 1)
    rows = _rows(1, *HEADS, torch.float16, seed=7)
    assert torch.equal(_run(other, turned, rows), _run(layer, step, rows))
    assert all(torch.equal(a, b) for a, b in zip(_bits(layer), _bits(other)))
    assert _native.device_error() == 0
