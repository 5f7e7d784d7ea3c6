"""Speculative decoding over an 8-bit K/V cache.

    PYTHONPATH=. python examples/speculative_kv8.py [--code e4m3] [--requests 4] [--tokens 96]
                                                    [--drafts 7] [--temperature 0.0]

Each step drafts tokens for every request by looking up the last two tokens in
what the request has so far, runs the model once over last token and drafts
(``B200KV8AttentionBackend``: the step's keys and values go into the 8-bit cache
with the rotation, then attention reads it), and lets ``verify_drafts`` accept
drafts and draw the next token.  A refused draft's slots are simply written over
by the next step.  The model is a small Qwen2 AWQ stack with random weights.
"""

from __future__ import annotations

import argparse
import time
from types import SimpleNamespace

import torch

from light_vllm_b200 import B200KV8AttentionBackend, KV8Cache, KV8CacheConfig, verify_drafts
from light_vllm_b200.qwen2 import Qwen2AWQRunner, Qwen2Shape, random_shard

CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def lookup_drafts(tokens: list[int], count: int, ngram: int = 2) -> list[int]:
    """Up to ``count`` tokens that followed the latest earlier occurrence of the
    last ``ngram`` tokens."""

    tail = tokens[-ngram:]
    for at in range(len(tokens) - ngram - 1, -1, -1):
        if tokens[at:at + ngram] == tail:
            return tokens[at + ngram:at + ngram + count]
    return []


def step_metadata(tables: list[list[int]], computed: list[int], lengths: list[int], block_size: int) -> SimpleNamespace:
    """The fields of light-vllm's ``PagedAttentionMetadata`` that a backend reads."""

    used = tuple(tuple(t[:-(-(c + n) // block_size)]) for t, c, n in zip(tables, computed, lengths))
    return SimpleNamespace(
        block_tables=used, num_computed_tokens=tuple(computed),
        query_layouts=tuple(SimpleNamespace(parent_indices=tuple(range(-1, n - 1))) for n in lengths),
        num_reserved_query_tokens=tuple(lengths), num_readonly_prefix_blocks=(0,) * len(lengths))


def probabilities(logits: torch.Tensor, temperature: float) -> torch.Tensor:
    """fp32 target probabilities; temperature 0 puts all of it on the greedy token."""

    if temperature == 0.0:
        return torch.zeros(logits.shape, device=logits.device).scatter_(1, logits.argmax(1, keepdim=True), 1.0)
    return torch.softmax(logits.float() / temperature, dim=1)


def generate(runner: Qwen2AWQRunner, cache: KV8Cache, prompts: list[list[int]], new_tokens: int, *, max_drafts: int,
             temperature: float, seed: int = 0) -> tuple[list[list[int]], dict[str, int]]:
    """``new_tokens`` tokens for every prompt, and counts of steps, drafts and
    accepted drafts.  A prompt's step must fit ``runner.max_tokens``."""

    device = runner.device
    longest = max(map(len, prompts), default=0) + new_tokens
    if longest - 1 > runner.shape.max_position_embeddings:  # (the last token is not run)
        raise ValueError(f"the model has {runner.shape.max_position_embeddings} positions, {longest - 1} are needed")
    backend = B200KV8AttentionBackend()
    uniform = torch.Generator(device=device).manual_seed(seed)
    block = cache.config.block_size
    need = [-(-(len(p) + new_tokens + max_drafts) // block) for p in prompts]
    if sum(need) > cache.config.num_blocks:
        raise ValueError(f"the cache holds {cache.config.num_blocks} blocks, {sum(need)} are needed")
    tables, at = [], 0
    for blocks in need:
        tables.append(list(range(at, at + blocks)))
        at += blocks

    tokens = [list(p) for p in prompts]
    computed = [0] * len(prompts)
    stats = {"steps": 0, "drafted": 0, "accepted": 0}
    while True:
        active = [r for r, t in enumerate(tokens) if len(t) < len(prompts[r]) + new_tokens]
        if not active:
            return tokens, stats
        # A request's first step is its prompt, every later one its last token; drafts follow.
        drafts = [lookup_drafts(tokens[r], min(max_drafts, len(prompts[r]) + new_tokens - len(tokens[r]) - 1))
                  if computed[r] else [] for r in active]
        ids = [tokens[r][computed[r]:] + d for r, d in zip(active, drafts)]
        lengths = [len(i) for i in ids]
        context = backend.create(cache, step_metadata([tables[r] for r in active], [computed[r] for r in active],
                                                      lengths, block))
        positions = torch.tensor([computed[r] + j for r, n in zip(active, lengths) for j in range(n)],
                                 dtype=torch.int32, device=device)
        # Of a request's rows, the last committed token's and its drafts' are verified.
        starts, rows, packed = 0, [], [0]
        for n, d in zip(lengths, drafts):
            rows += range(starts + n - 1 - len(d), starts + n)
            packed.append(len(rows))
            starts += n
        logits = runner.logits(torch.tensor([i for r in ids for i in r], device=device), positions, context,
                               torch.tensor(rows, device=device))
        flat = [i for d in drafts for i in d]
        out, accepted = verify_drafts(
            probabilities(logits, temperature), torch.tensor(flat, dtype=torch.int64, device=device),
            torch.rand(len(flat), device=device, generator=uniform),
            torch.rand(len(active), device=device, generator=uniform),
            torch.tensor(packed, dtype=torch.int32, device=device), max_query_len=max(map(len, drafts)) + 1)
        for r, d, row, kept in zip(active, drafts, out.tolist(), accepted.tolist()):
            computed[r] = len(tokens[r]) + kept
            tokens[r] += row[:kept + 1]
            stats["drafted"] += len(d)
            stats["accepted"] += kept
        stats["steps"] += 1


def demo_prompts(requests: int) -> list[list[int]]:
    """Prompts of 16, 21, .. tokens."""

    return [[(r * 31 + j * j) % 512 for j in range(16 + 5 * r)] for r in range(requests)]


def step_tokens(prompts: list[list[int]], max_drafts: int) -> int:
    """Tokens of ``generate``'s longest step: all prompts, or every request's last token and drafts."""

    return max(sum(map(len, prompts)), len(prompts) * (max_drafts + 1))


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--code", choices=sorted(CODES), default="int8")
    parser.add_argument("--requests", type=int, default=4)
    parser.add_argument("--tokens", type=int, default=96)
    parser.add_argument("--drafts", type=int, default=7)
    parser.add_argument("--temperature", type=float, default=0.0)
    args = parser.parse_args()
    device = torch.device("cuda", 0)
    shape = Qwen2Shape(vocab_size=512, hidden_size=256, intermediate_size=512, num_hidden_layers=2,
                       num_attention_heads=4, num_key_value_heads=2, max_position_embeddings=2048)
    weights = random_shard(shape, 0, 1, device)
    # The last token then weighs most in the next one, so that the output repeats itself and drafts are found.
    weights["model.embed_tokens.weight"] *= 500
    prompts = demo_prompts(args.requests)
    runner = Qwen2AWQRunner(shape, weights, device, max_tokens=step_tokens(prompts, args.drafts))
    blocks = sum(-(-(len(p) + args.tokens + args.drafts) // 16) for p in prompts)
    try:
        for drafts in (0, args.drafts):
            cache = KV8Cache(runner.kv_layers(), KV8CacheConfig(blocks, 16, CODES[args.code], device))
            generate(runner, cache, prompts, 8, max_drafts=drafts, temperature=args.temperature)  # warm-up
            begin = time.perf_counter()
            tokens, stats = generate(runner, cache, prompts, args.tokens, max_drafts=drafts, temperature=args.temperature)
            took = time.perf_counter() - begin
            print(f"{drafts} drafts: {stats['steps']} steps, {stats['accepted']} of {stats['drafted']} drafts accepted, "
                  f"{args.requests * args.tokens / took:.0f} tokens/s; request 0 ends in {tokens[0][-8:]}")
    finally:
        torch.cuda.synchronize()
        runner.close()


if __name__ == "__main__":
    main()
