"""sample_tokens where a row is cut over several workgroups (few long rows): the
same definition, the same exact tokens."""

from __future__ import annotations

import math

import pytest
import torch

from mini_llm_runtime_amd import _lib
from mini_llm_runtime_amd.kernels.sampling import sample_tokens
from test_gpu_sampling import check, logits_of, uniforms_of

pytestmark = pytest.mark.gpu

VOCAB = 130003  # odd: rows start at every alignment


def test_rows_are_cut(device):
    assert _lib.load().mlr_sample_tokens_workspace_size(8, VOCAB) > 0


@pytest.mark.parametrize("params", [{}, {"top_k": 10}, {"top_k": 3000}, {"top_p": 0.5},
                                    {"min_p": 0.01}, {"temperature": 0.0}], ids=str)
def test_masked_infinite_and_missing_values(device, params):
    x = logits_of(device, 8, VOCAB, torch.float32, seed=41)
    x[0] = -math.inf
    x[1, :-1] = -math.inf
    x[2, ::2] = -math.inf
    x[3, ::3] = math.nan
    x[4] = math.nan
    x[5, 70000:70003] = math.inf
    x[6] = torch.finfo(torch.float32).min
    x[7, 5] = torch.finfo(torch.float32).max
    got = check(x, uniforms_of(8, 42), **params)
    assert got[0] == -1 and got[4] == -1 and got[1] == VOCAB - 1 and got[5] == 70000


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("params", [{}, {"top_k": 3000}, {"top_k": 100000, "top_p": 0.97},
                                    {"temperature": 50.0, "top_p": 0.4, "min_p": 0.1},
                                    {"temperature": math.inf}, {"temperature": 1e-40}], ids=str)
def test_crowded_bins(device, dtype, params):
    """More values in a bin than a list holds, in every part of the row."""
    gen = torch.Generator().manual_seed(43)
    x = (1.0 + torch.randint(0, 60, (5, VOCAB), generator=gen) * 2.0 ** -23).to(device)
    x[:, 99991] = 8.0
    x[3] += 1e-3 * torch.randn(VOCAB, generator=gen).to(device)
    x[4] = -2.0
    check(x.to(dtype), torch.tensor([0.1, 0.5, 0.999, 0.3, 0.7]), **params)


def test_rows_strides_and_parameters_of_each_row(device):
    x = logits_of(device, 6, VOCAB + 9, torch.float16, seed=44)[:, 5:VOCAB + 5]
    rows = torch.tensor([5, 0, 5, 2])
    check(x, uniforms_of(4, 45), rows=rows,
          temperature=torch.tensor([0.0, 0.7, 1.0, 2.5]), top_k=torch.tensor([0, 2049, 1, 60]),
          top_p=torch.tensor([0.9, 0.8, 0.5, 1.0]), min_p=torch.tensor([0.0, 0.0, 0.1, 0.02]))
    got = sample_tokens(x, uniforms_of(4, 46).to(device),
                        rows=torch.tensor([0, -1, 6, 2 ** 40], device=device))
    assert got[1:].tolist() == [-1, -1, -1] and got[0] >= 0


def test_two_graphs_replayed_in_turn(device):
    x = [logits_of(device, 3, VOCAB, torch.float32, seed=47 + i) for i in range(2)]
    u = uniforms_of(3, 49).to(device)
    want = [sample_tokens(v, u, top_p=0.9) for v in x]
    graphs, outs = [], []
    for v in x:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(sample_tokens(v, u, top_p=0.9))
        graphs.append(g)
    for _ in range(3):
        for o in outs:
            o.fill_(-7)
        for g in (graphs[0], graphs[1], graphs[0]):
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
