"""Decode over a shared prefix on both sides of the batch from which the requests' own
keys go to a launch of their own."""

from __future__ import annotations

import pytest
import torch

from test_gpu_scored_attention import shared_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv", [(12, 4), (14, 14)])
def test_large_batches(device, dtype, hq, hkv):
    most = 4 * torch.cuda.get_device_properties(device).multi_processor_count // hkv
    for batch in (most, most + 1):
        shared_case(device, 90, [(5 * i) % 37 for i in range(batch)], hq, hkv, 64, 16, dtype,
                    dict(cap=20.0))
