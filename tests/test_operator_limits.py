"""Sizes, ranges and empty calls of the operators at their ends, on the CPU: nothing
here reaches a GPU."""

from __future__ import annotations

import math

import pytest
import torch

from mini_llm_runtime_amd import _lib
from mini_llm_runtime_amd.kernels.pre_attention import rotary_frequencies

MB = 1 << 20


@pytest.mark.parametrize("batch,hq,hkv,most", [
    (1024, 32, 32, 160), (256, 12, 12, 64), (4096, 4, 4, 160), (32, 32, 32, 64), (64, 14, 2, 64)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_shared_prefix_workspace(batch, hq, hkv, most, dtype):
    """Partial results of 16 rows a request and KV head where there are many of them
    (4.2 KB at head size 64), and of 128 rows for some two thousand at most."""
    size = _lib.load().mlr_paged_decode_shared_prefix_workspace_size(
        batch, hq, hkv, 64, 8192, 576, 16, _lib.DTYPE_CODES[dtype])
    assert 0 < size <= most * MB


@pytest.mark.parametrize("dtype,block_size", [(torch.float32, 16), (torch.bfloat16, 24)])
@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (32, 8, 128)])
def test_prefill_workspace(dtype, block_size, hq, hkv, d):
    """One long prompt in a batch of many sequences does not reserve partial results
    for as many long ones."""
    size = _lib.load().mlr_paged_prefill_scored_workspace_size
    code = _lib.DTYPE_CODES[dtype]
    for seqs in (1, 8, 64, 1000):
        for longest in (1, 16, 512, 4096, 32768):
            assert size(seqs, longest, 4096, block_size, hq, hkv, d, code) <= 256 * MB
    assert size(8, 512, 4096, block_size, hq, hkv, d, code) > 0


@pytest.mark.parametrize("base", [1.0, 0.5])
def test_yarn_needs_falling_frequencies(base):
    with pytest.raises(ValueError, match="base above 1"):
        rotary_frequencies(8, base, scaling="yarn", factor=2.0, original_max_position=64)
    freq, m = rotary_frequencies(8, 1.0, scaling="ntk", factor=8.0)
    assert m == 1.0 and abs(float(freq[-1]) * 8.0 - 1.0) < 1e-6


@pytest.mark.parametrize("scaling", ["linear", "ntk", "yarn"])
def test_factor_must_be_finite(scaling):
    with pytest.raises(ValueError, match="factor"):
        rotary_frequencies(8, scaling=scaling, factor=math.inf, original_max_position=64)
