"""Scored prefill of a batch with room for far more rows than it has: its units stay
whole, as partial results of all that room would take too much memory."""

from __future__ import annotations

import pytest
import torch

from mini_llm_runtime_amd import _lib
from mini_llm_runtime_amd.kernels.scored_attention import paged_attention_prefill_scored
from test_gpu_scored_attention import prefill_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,bs", [(torch.float32, 16), (torch.bfloat16, 24)])
def test_one_long_prompt_among_many(device, dtype, bs):
    chunks = [(0, 0)] * 150 + [(3, 40), (700, 90), (0, 900), (2000, 1)] + [(5, 1)] * 150
    size = _lib.load().mlr_paged_prefill_scored_workspace_size
    assert size(len(chunks), 900, 130, bs, 14, 1, 64, _lib.DTYPE_CODES[dtype]) == 0
    prefill_case(device, chunks, 14, 1, 64, bs, dtype, dict(cap=20.0, alibi=True))


def test_metadata_of_empty_batches_is_checked(device):
    """Tokens without a sequence, and sequences that claim tokens that are not there."""
    k = torch.zeros(3, 16, 2, 64, dtype=torch.bfloat16, device=device)

    def call(tokens, qsl, ctx, width=2):
        q = torch.zeros(tokens, 4, 64, dtype=torch.bfloat16, device=device)
        return paged_attention_prefill_scored(
            q, k, k, torch.zeros(len(ctx), width, dtype=torch.long, device=device),
            torch.tensor(qsl, device=device), torch.tensor(ctx, dtype=torch.long, device=device),
            16)

    assert call(0, [0], []).shape == (0, 4, 64)
    assert call(0, [0, 0, 0], [5, 0]).shape == (0, 4, 64)
    for args, needle in [((7, [0], []), "end at the packed"), ((0, [0, 3], [9]), "end at the packed"),
                         ((0, [0, 0], [90]), "insufficient blocks"), ((0, [1], []), "start at 0")]:
        with pytest.raises(ValueError, match=needle):
            call(*args)
