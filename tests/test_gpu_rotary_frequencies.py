"""Rotary frequencies that are not in FP32: calls that a graph records first, and
buffers changed between calls."""

from __future__ import annotations

import pytest
import torch

from mini_llm_runtime_amd.kernels.pre_attention import qk_norm_rope_write
from test_gpu_qk_norm_rope import check, make

pytestmark = pytest.mark.gpu


def other_dtype(device, seed):
    t = make(device, 17, 4, 2, 64, 64, torch.bfloat16, seed=seed)
    t["inv_freq"] = t["inv_freq"].bfloat16()
    return t


def test_recorded_before_any_eager_call(device):
    """The eager call after the capture and before a replay has the frequencies too."""
    t = other_dtype(device, 20)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = qk_norm_rope_write(t["qkv"], t["positions"], t["inv_freq"], t["k"], t["v"],
                                 t["slots"], 4, q_weight=t["qw"], k_weight=t["kw"])
    want = check(t, 4, 2, 64)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_frequencies_changed_in_place(device):
    t = other_dtype(device, 21)
    check(t, 4, 2, 64)
    t["inv_freq"].mul_(0.5)
    check(t, 4, 2, 64)
    t["inv_freq"].data.mul_(0.25)  # leaves the version as it is
    check(t, 4, 2, 64)


def test_inference_tensors(device):
    with torch.inference_mode():
        t = other_dtype(device, 22)
        check(t, 4, 2, 64)
