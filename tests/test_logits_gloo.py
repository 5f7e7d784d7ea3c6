"""``Qwen2AWQRunner.logits`` over vocabulary shards, equal and unequal, on gloo CPU ranks."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch
import torch.multiprocessing as mp

from light_vllm_b200.collectives import partition_dimension
from light_vllm_b200.qwen2 import Qwen2AWQRunner
from test_tensor_parallel_gloo import _free_port, _init

HIDDEN, ROWS = 16, 5


def _whole(vocab):
    gen = torch.Generator().manual_seed(vocab)
    return torch.randn((vocab, HIDDEN), generator=gen), torch.randn((ROWS, HIDDEN), generator=gen)


def _worker(rank, world, port, vocab, results):
    _init(rank, world, port, 60)
    head, hidden = _whole(vocab)
    part = partition_dimension(vocab, rank, world)
    runner = Qwen2AWQRunner.__new__(Qwen2AWQRunner)  # the head and its gather need nothing of the stack
    runner.rank, runner.world, runner.group, runner.device = rank, world, None, torch.device("cpu")
    runner.layout = SimpleNamespace(vocab_part=part)
    runner.lm_head = head[part.start:part.end].contiguous()
    runner._hidden = lambda *args: hidden
    try:
        results.put((rank, runner.logits(None, None, None).numpy()))
    finally:
        torch.distributed.destroy_process_group()


@pytest.mark.parametrize("world,vocab", [(2, 64), (2, 65), (3, 65), (3, 64)])
def test_logits_of_every_rank(world, vocab):
    context = mp.get_context("spawn")
    results, port = context.Queue(), _free_port()
    ranks = [context.Process(target=_worker, args=(r, world, port, vocab, results)) for r in range(world)]
    for p in ranks:
        p.start()
    try:
        got = dict(results.get(timeout=90) for _ in ranks)
    finally:
        for p in ranks:
            p.join(30)
            if p.is_alive():
                p.terminate()
    head, hidden = _whole(vocab)
    want = hidden @ head.t()
    for logits in got.values():
        assert logits.shape == want.shape
        assert torch.allclose(torch.from_numpy(logits), want, rtol=1e-5, atol=1e-4)  # fp32 sums of 16 products of normal values
