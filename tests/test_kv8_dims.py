"""Arguments of too few dimensions are refused with the operators' own messages (CPU only)."""

from __future__ import annotations

import pytest
import torch

from light_vllm_b200 import KV8Step, KVCacheError, verify_drafts
from light_vllm_b200.kv8 import _check_rows, _check_step

INT = dict(dtype=torch.int32)
GOOD = KV8Step(torch.zeros((1, 1), **INT), torch.zeros(1, **INT), torch.zeros(2, **INT), 1, 1)


@pytest.mark.parametrize("field", ["block_tables", "num_computed", "query_start"])
def test_step_metadata_of_no_dimensions(field):
    with pytest.raises(KVCacheError, match="int32"):
        _check_step(GOOD._replace(**{field: torch.tensor(0, **INT)}), -1)


def test_rows_of_no_dimensions():
    with pytest.raises(KVCacheError, match=r"\[tokens, heads, head_size\]"):
        _check_rows("key", torch.tensor(0.0).half(), None, 2, 64, torch.float16, -1)


@pytest.mark.parametrize("name", ["draft_tokens", "accept_uniform", "sample_uniform"])
def test_drafts_of_no_dimensions(name, monkeypatch):
    args = dict(draft_tokens=torch.zeros(2, dtype=torch.int64), accept_uniform=torch.zeros(2), sample_uniform=torch.zeros(1),
                query_start=torch.zeros(2, **INT))
    args[name] = args[name].new_zeros(())
    monkeypatch.setattr(torch.Tensor, "get_device", lambda self: 0)
    with pytest.raises(ValueError, match="one uniform number for each draft"):
        verify_drafts(torch.zeros((3, 8)), **args, max_query_len=3)
