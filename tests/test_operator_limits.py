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
