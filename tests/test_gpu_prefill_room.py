"""Scored prefill of a batch with room for far more rows than it has: its units stay
whole, as partial results of all that room would take too much memory."""

from __future__ import annotations

import pytest
import torch

from mini_llm_runtime_amd import _lib
from test_gpu_scored_attention import prefill_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,bs", [(torch.float32, 16), (torch.bfloat16, 24)])
def test_one_long_prompt_among_many(device, dtype, bs):
    chunks = [(0, 0)] * 150 + [(3, 40), (700, 90), (0, 900), (2000, 1)] + [(5, 1)] * 150
    size = _lib.load().mlr_paged_prefill_scored_workspace_size
    assert size(len(chunks), 900, 130, bs, 14, 1, 64, _lib.DTYPE_CODES[dtype]) == 0
    prefill_case(device, chunks, 14, 1, 64, bs, dtype, dict(cap=20.0, alibi=True))
