"""Rotary frequencies that are not in FP32: calls that a graph records first, and
buffers changed between calls."""

from __future__ import annotations

import pytest
import torch

from mini_llm_runtime_amd.kernels.pre_attention import qk_norm_rope_write, qkv_rope_write
from mini_llm_runtime_amd.runtime.paged_kv_cache import PagedKVCache
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


def plain_call(t, cache):
    return qkv_rope_write(t["qkv"], t["positions"], t["inv_freq"], cache, 0, t["slots"], 4)


def test_plain_append_recorded_before_any_eager_call(device):
    t = other_dtype(device, 23)
    cache = PagedKVCache(1, t["k"].shape[0], 16, 2, 64, dtype=torch.bfloat16, device=device)
    want = plain_call(dict(t, inv_freq=t["inv_freq"].float()), cache)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = plain_call(t, cache)
    assert torch.equal(plain_call(t, cache), want)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    with torch.inference_mode():
        assert torch.equal(plain_call(dict(t, inv_freq=t["inv_freq"].clone()), cache), want)


def test_copies_outlive_the_cache(device):
    """A graph that recorded a kept copy replays rightly after the copy left the cache."""
    t = other_dtype(device, 24)
    cache = PagedKVCache(1, t["k"].shape[0], 16, 2, 64, dtype=torch.bfloat16, device=device)
    want = plain_call(t, cache)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = plain_call(t, cache)
    others = [torch.full((32,), float(i), dtype=torch.bfloat16, device=device) for i in range(70)]
    for f in others:
        plain_call(dict(t, inv_freq=f), cache)
    fill = [torch.full((32,), 7.0, device=device) for _ in range(200)]
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert len(fill) == 200
