"""Verification of drafted tokens by speculative sampling.

``verify_drafts`` accepts or refuses a step's drafted tokens against the
target model's probabilities, and draws the token that follows the accepted
ones, from uniform numbers that the caller gives (``lvb_verify_drafts``).  The
emitted tokens follow the target's distribution, whatever drafted them, in the
steps of the uniform numbers: fp32 ones from a generator are multiples of 2^-24,
so a token of less probability is drawn with probability 0 or 2^-24.  The reference accepts drafts by greedy comparison only
(runtime/execution/speculative.py); target probabilities that are 1 at the
greedy token give that rule.
"""

from __future__ import annotations

import torch
from torch import Tensor

from light_vllm_b200 import _native
from light_vllm_b200.kv8 import _on, _Workspaces

_workspaces = _Workspaces(1)
_fast = None  # _torch_ops, loaded by the first call


def verify_drafts(target_probs: Tensor, draft_tokens: Tensor, accept_uniform: Tensor, sample_uniform: Tensor,
                  query_start: Tensor, *, max_query_len: int,
                  draft_probs: Tensor | None = None) -> tuple[Tensor, Tensor]:
    """Returns (tokens int64 [requests, max_query_len], accepted int32
    [requests]): each request's accepted drafts, then the drawn token, then -1.

    The packing is the verification step's own.  Request b's query rows
    ``query_start[b] .. query_start[b + 1]`` (its last committed token, then
    its drafts) give its rows of ``target_probs`` [rows, vocabulary] fp32;
    ``draft_tokens`` (int64), ``accept_uniform`` (fp32) and ``draft_probs``
    [drafts, vocabulary] (fp32) hold the drafts of all requests, so one row
    fewer for each.  ``sample_uniform`` is fp32, one for each request.  Without
    ``draft_probs`` the drafts were looked up rather than drawn, and draft x is
    accepted with probability p(x).  ``max_query_len`` is the longest request's
    row count."""

    global _fast
    if _fast is None:
        _fast = _native.torch_ops()
    done = _fast.verify_drafts(target_probs, draft_tokens, accept_uniform, sample_uniform, query_start, max_query_len,
                               draft_probs)
    if done is not None:
        if type(done) is int:
            _native.check(done, "lvb_verify_drafts")
        return done

    if target_probs.dtype != torch.float32 or target_probs.dim() != 2:
        raise ValueError("target probabilities must be float32 [rows, vocabulary]")
    index = target_probs.get_device()
    if index < 0:
        raise ValueError("draft verification runs on a CUDA device")
    rows, vocab = target_probs.shape
    if vocab == 0:
        raise ValueError("the vocabulary must not be empty")
    if query_start.dtype != torch.int32 or query_start.dim() != 1 or query_start.shape[0] == 0:
        raise ValueError("query_start must be an int32 vector of requests + 1 values")
    n, drafts = query_start.shape[0] - 1, draft_tokens.numel()
    if draft_tokens.dtype != torch.int64 or accept_uniform.dtype != torch.float32 or sample_uniform.dtype != torch.float32:
        raise ValueError("draft tokens must be int64 and uniform numbers float32")
    if draft_tokens.dim() != 1 or accept_uniform.shape != draft_tokens.shape or sample_uniform.shape != (n,):
        raise ValueError("one uniform number for each draft and one for each request are required")
    if draft_probs is not None and (draft_probs.dtype != torch.float32 or draft_probs.shape != (drafts, vocab)):
        raise ValueError("draft probabilities must be float32 [drafts, vocabulary]")
    if max_query_len < 0 or rows != drafts + n:
        raise ValueError("target probabilities must have one row for each draft and one more for each request")
    for t in (draft_tokens, accept_uniform, sample_uniform, query_start):
        if t.get_device() != index or not t.is_contiguous():
            raise ValueError("draft tokens, uniform numbers and query_start must be contiguous on one device")
    if draft_probs is not None and draft_probs.get_device() != index:
        raise ValueError("draft probabilities must be on the target probabilities' device")
    target_probs, target_stride = _dense_rows(target_probs)
    draft_ptr = draft_stride = 0
    if draft_probs is not None and drafts:
        draft_probs, draft_stride = _dense_rows(draft_probs)
        draft_ptr = draft_probs.data_ptr()
    device = target_probs.device
    tokens = torch.empty((n, max_query_len), dtype=torch.int64, device=device)
    accepted = torch.empty(n, dtype=torch.int32, device=device)
    if n:
        with _on(index):
            lib = _native.library()
            stream = _native.stream_handle(device)
            ws, ws_bytes = _workspaces.get(device, stream, lib.lvb_verify_drafts_workspace_bytes(n, vocab))
            _native.check(lib.lvb_verify_drafts(
                target_probs.data_ptr(), target_stride, draft_ptr, draft_stride, draft_tokens.data_ptr(),
                accept_uniform.data_ptr(), sample_uniform.data_ptr(), query_start.data_ptr(), tokens.data_ptr(),
                accepted.data_ptr(), n, rows, max_query_len, vocab, ws, ws_bytes, stream), "lvb_verify_drafts")
    return tokens, accepted


def _dense_rows(probs: Tensor) -> tuple[Tensor, int]:
    """Rows whose values are dense, and their stride."""

    rows, vocab = probs.shape
    if (vocab > 1 and probs.stride(1) != 1) or (rows > 1 and probs.stride(0) < vocab):
        probs = probs.contiguous()
    return probs, probs.stride(0) if rows > 1 else vocab
