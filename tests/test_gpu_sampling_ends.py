"""sample_tokens at the ends of what its parameters may be: temperatures next to 0 and
without bound, against the definition."""

from __future__ import annotations

import math

import pytest
import torch

from mini_llm_runtime_amd.kernels.sampling import sample_tokens
from test_gpu_sampling import check, logits_of, uniforms_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("params", [{}, {"top_k": 7}, {"top_k": 3000}, {"top_p": 0.5},
                                    {"min_p": 1.0}, {"min_p": 0.3, "top_p": 0.7}], ids=str)
@pytest.mark.parametrize("temperature", [5e-324, 1e-310, 1e-300, 1e-45, 1e300, 1.7e308, math.inf,
                                         torch.tensor([1e-45, math.inf] * 3)], ids=str)
@pytest.mark.parametrize("dtype,vocab", [(torch.float32, 1000), (torch.float32, 5003),
                                         (torch.bfloat16, 5003), (torch.float32, 130003),
                                         (torch.bfloat16, 130003)])
def test_temperatures(device, dtype, vocab, temperature, params):
    x = logits_of(device, 6, vocab, dtype, seed=91)
    top = x.amax(1)
    x[:, 17] = x[:, 900] = top  # a draw between equal ones where all else weighs 0
    x[4:, 30] = top[4:].float().abs().to(dtype) * 2
    check(x, uniforms_of(6, 92), temperature=temperature, **params)


@pytest.mark.parametrize("vocab", [1000, 130003])
def test_no_logits_rows_at_all(device, vocab):
    """Every row id is out of range then."""
    tokens, logprobs = sample_tokens(torch.empty(0, vocab, device=device),
                                     torch.full((3,), 0.5, device=device), return_logprobs=True,
                                     rows=torch.tensor([0, -1, 7], device=device))
    assert tokens.tolist() == [-1] * 3 and logprobs.tolist() == [-math.inf] * 3
