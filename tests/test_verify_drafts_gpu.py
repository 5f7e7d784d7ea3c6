"""Draft verification on the GPU: equal to the rule in whole numbers, draw for draw."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from light_vllm_b200 import _native, verify_drafts
from oracle import speculative as ospec

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def _dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).to(DEV)


def _case(drafts, vocab, probs, seed, peak=4.0):
    rng = np.random.default_rng(seed)
    rows, total = sum(drafts) + len(drafts), sum(drafts)

    def soft(x):
        e = np.exp(x - x.max(axis=1, keepdims=True))
        return (e / e.sum(axis=1, keepdims=True)).astype(np.float32)

    logits = rng.standard_normal((rows, vocab)) * peak
    start = np.cumsum([0] + [k + 1 for k in drafts]).astype(np.int32)
    at = np.array([start[b] + i for b, k in enumerate(drafts) for i in range(k)], dtype=int)
    target = soft(logits)
    draft = soft(logits[at] + rng.standard_normal((total, vocab)) * 0.7) if probs and total else None
    source = draft if draft is not None else soft(2.0 * logits[at]) if total else np.zeros((0, vocab))
    tokens = np.array([rng.choice(vocab, p=p.astype(np.float64) / p.astype(np.float64).sum()) for p in source], dtype=np.int64)
    return (target, tokens, rng.random(total, dtype=np.float32), rng.random(len(drafts), dtype=np.float32), start, draft)


def _run(target, tokens, accept, sample, start, draft, width):
    return verify_drafts(_dev(target), _dev(tokens), _dev(accept), _dev(sample), _dev(start), max_query_len=width,
                         draft_probs=None if draft is None else _dev(draft))


def _check(case, width=None):
    target, tokens, accept, sample, start, draft = case
    width = int(np.diff(start).max()) if width is None else width
    got = _run(*case, width)
    want = ospec.verify(target, tokens, accept, sample, start, width, draft)
    assert (got[0].cpu().numpy() == want[0]).all()
    assert (got[1].cpu().numpy() == want[1]).all()
    assert _native.device_error() == 0
    return got


@pytest.mark.parametrize("probs", [True, False])
@pytest.mark.parametrize("vocab", [1, 2, 31, 1000, 4097, 50257, 152064])
@pytest.mark.parametrize("drafts", [[0], [1], [4], [0, 3, 1, 0, 7, 2], [5] * 17, [40, 0, 33]], ids=lambda d: f"{len(d)}x{max(d)}")
def test_verification(drafts, vocab, probs):
    _check(_case(drafts, vocab, probs, seed=vocab + len(drafts)))


@pytest.mark.parametrize("probs", [True, False])
def test_many_requests(probs):
    rng = np.random.default_rng(1)
    _check(_case(rng.integers(0, 6, 400).tolist(), 777, probs, seed=2))


@pytest.mark.parametrize("sample", [0.0, 0.5, 1.0 - 2.0 ** -24])
def test_the_ends_of_the_uniform_range(sample):
    target, tokens, accept, _, start, draft = _case([2, 0, 3], 301, True, seed=3)
    for u in (0.0, 1.0 - 2.0 ** -24):
        accept[:] = u
        _check((target, tokens, accept, np.full(3, sample, np.float32), start, draft))
    target[:, :5] = 0  # leading and trailing tokens without mass are never drawn
    target[:, -5:] = 0
    got = _check((target, tokens, accept, np.full(3, sample, np.float32), start, None))
    for row, n in zip(got[0].cpu(), got[1].cpu()):
        assert 5 <= row[n] < 296


def test_rows_without_mass_and_values_that_are_no_probabilities():
    target, tokens, accept, sample, start, draft = _case([2, 2, 2, 1, 1], 515, True, seed=4)
    draft[:2] = target[:2]  # p = q: nothing left where it is refused
    accept[:2] = 1.0
    target[3:6] = 0  # a target without any mass
    target[6, ::2] = np.nan
    draft[4, ::3] = np.nan
    target[9, 7] = np.inf
    target[10, 100:] = -1.0
    target[11:] *= 3.0  # not normalised
    _check((target, tokens, accept, sample, start, draft))
    _check((target, tokens, accept, sample, start, None))


def test_no_requests():
    none = torch.zeros(0, device=DEV)
    got = verify_drafts(torch.zeros((0, 9), device=DEV), none.long(), none, none, _dev(np.zeros(1, np.int32)), max_query_len=0)
    assert got[0].shape == (0, 0) and got[1].shape == (0,)


def test_strided_and_unaligned_rows():
    case = _case([3, 1, 4], 1003, True, seed=6)
    want = _check(case)
    target, tokens, accept, sample, start, draft = case
    wide = torch.zeros((target.shape[0], 1203), device=DEV)
    wide[:, 101:1104] = _dev(target)
    wide_draft = torch.zeros((draft.shape[0], 2000), device=DEV)
    wide_draft[:, 7:1010] = _dev(draft)
    got = verify_drafts(wide[:, 101:1104], _dev(tokens), _dev(accept), _dev(sample), _dev(start), max_query_len=5,
                        draft_probs=wide_draft[:, 7:1010])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    turned = _dev(np.ascontiguousarray(target.T)).t()  # columns outermost: copied
    got = verify_drafts(turned, _dev(tokens), _dev(accept), _dev(sample), _dev(start), max_query_len=5, draft_probs=_dev(draft))
    assert torch.equal(got[0], want[0])


def test_a_draft_outside_the_vocabulary_is_refused_and_reported():
    target, tokens, accept, sample, start, draft = _case([2, 2], 64, True, seed=7)
    tokens[1], tokens[2] = 64, -1
    accept[:] = 0
    for d in (draft, None):
        got = _run(target, tokens, accept, sample, start, d, 3)
        assert _native.device_error() == 2
        want = ospec.verify(target, tokens, accept, sample, start, 3, d)
        assert (got[0].cpu().numpy() == want[0]).all() and got[1].tolist() == want[1].tolist() == [1, 0]


def test_rows_outside_the_batch_are_reported():
    """Rows that do not exist, no rows at all, more rows than named: -1 throughout, and the others stand."""

    case = _case([2, 2], 64, True, seed=8)
    target, tokens, accept, sample, start, draft = case
    want = _check(case)
    for bad, fine in (([0, 4, 6], None), ([0, 3, 8], 0), ([-1, 3, 6], 1), ([3, 3, 6], 1), ([0, 0, 3], None)):
        got = _run(target, tokens, accept, sample, np.array(bad, np.int32), draft, 3)
        assert _native.device_error() == 2
        for b in range(2):
            if b == fine:
                assert torch.equal(got[0][b], want[0][b]) and got[1][b] == want[1][b]
    got = _run(target, tokens, accept, sample, np.array([3, 3, 6], np.int32), draft, 3)
    assert _native.device_error() == 2
    assert got[0][0].tolist() == [-1, -1, -1] and got[1][0] == 0


@pytest.mark.parametrize("probs", [True, False])
def test_emitted_tokens_follow_the_target(probs):
    """The first token of 40000 requests of one draft each: within five standard deviations of p."""

    n, vocab = 40000, 8
    rng = np.random.default_rng(9)
    p = np.array([0.4, 0.05, 0.2, 0.01, 0.14, 0.1, 0.1, 0.0], np.float32)
    q = np.array([0.1, 0.3, 0.2, 0.05, 0.05, 0.1, 0.1, 0.1], np.float32)
    target = np.tile(p, (2 * n, 1))
    draft = np.tile(q, (n, 1)) if probs else None
    tokens = rng.choice(vocab, n, p=q.astype(np.float64) / q.astype(np.float64).sum()).astype(np.int64)
    got = _run(target, tokens, rng.random(n, dtype=np.float32), rng.random(n, dtype=np.float32),
               np.arange(0, 2 * n + 1, 2, dtype=np.int32), draft, 2)
    count = np.bincount(got[0][:, 0].cpu().numpy(), minlength=vocab)
    assert (np.abs(count - n * p) <= 5 * np.sqrt(n * p * (1 - p)) + 1e-6).all()
    second = got[0][:, 1].cpu().numpy()
    taken = got[1].cpu().numpy() == 1
    assert (second[~taken] == -1).all()
    count, m = np.bincount(second[taken], minlength=vocab), taken.sum()
    assert (np.abs(count - m * p) <= 5 * np.sqrt(m * p * (1 - p)) + 1e-6).all()


@pytest.mark.parametrize("kind", ["halves", "small", "steps", "wide", "ones"])
def test_weights_become_whole_numbers_by_the_rule(kind):
    """Draws from weights whose whole numbers show how they were rounded."""

    rng = np.random.default_rng(7)
    rows, vocab = 96, 5000
    if kind == "halves":  # ties: to the even neighbour
        target = (rng.integers(0, 64, (rows, vocab)) + 0.5) * 2.0 ** -40
    elif kind == "small":  # around half of the least weight, and far below
        target = np.exp2(rng.uniform(-60, -38, (rows, vocab)))
    elif kind == "steps":  # at the multiples of 2^-20 where the parts of a weight meet
        target = (rng.integers(0, 9, (rows, vocab)) + rng.choice([-0.5, 0.0, 0.5], (rows, vocab))) * 2.0 ** -20
        target = np.abs(target + rng.integers(-3, 4, (rows, vocab)) * 2.0 ** -40)
    elif kind == "wide":
        target = np.exp2(rng.uniform(-45, 0, (rows, vocab)))
    else:
        target = np.ones((rows, vocab))
    target = target.astype(np.float32)
    none = np.zeros(0, np.float32)
    start = np.arange(rows + 1, dtype=np.int32)
    _check((target, np.zeros(0, np.int64), none, rng.random(rows, dtype=np.float32), start, None))
