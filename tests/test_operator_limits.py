"""Sizes, ranges and empty calls of the operators at their ends, on the CPU: nothing
here reaches a GPU."""

from __future__ import annotations

import pytest
import torch

from mini_llm_runtime_amd import _lib

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
