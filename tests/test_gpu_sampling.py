"""sample_tokens (mlr_sample_tokens) against its definition in 64 bits.

Tokens must be equal: the kernel's weights are within 7e-12 of the exact ones
and within 2^-45 of the largest, so a drawn target would have to fall within
about 1e-11 of a border for the two to differ. Log-probabilities: one FP32
rounding of a value whose argument is exact to 1e-11, so 2^-24 |l| + 1e-9.
"""

from __future__ import annotations

import math

import pytest
import torch

from mini_llm_runtime_amd.kernels.sampling import sample_tokens

pytestmark = pytest.mark.gpu


def definition(x, u, t=1.0, k=0, p=1.0, m=0.0):
    """(token, logprob) of one row, on the CPU in 64 bits."""
    x = x.double().cpu()
    x = torch.where(x.isnan(), -math.inf, x)
    order = torch.argsort(x, descending=True, stable=True)
    top = float(x[order[0]])
    if top == -math.inf:
        return -1, -math.inf
    if not t > 0 or top == math.inf:
        return int(order[0]), 0.0
    w = torch.exp((x[order] - top) / t)
    n = len(w) if k <= 0 else min(k, len(w))
    mass = w[:n].cumsum(0)
    if p < 1:
        n = min(n, int((mass < p * mass[-1]).sum()) + 1) if p > 0 else 1
    if m > 0:
        n = min(n, max(1, int((w >= m).sum())))
    mass = w[:n].cumsum(0)
    at = min(int((mass <= u * float(mass[-1])).sum()), n - 1)
    while w[at] == 0:
        at -= 1
    return int(order[at]), math.log(float(w[at] / mass[-1]))


def check(logits, uniforms, rows=None, **params):
    """Whole call against the definition, row by row."""
    device = logits.device
    b = uniforms.shape[0]
    args = {n: v.to(device) if isinstance(v, torch.Tensor) else v for n, v in params.items()}
    got, logprob = sample_tokens(logits, uniforms.to(device), return_logprobs=True,
                                 rows=None if rows is None else rows.to(device), **args)
    short = {"temperature": "t", "top_k": "k", "top_p": "p", "min_p": "m"}
    for r in range(b):
        at = {short[n]: v[r].item() if isinstance(v, torch.Tensor) else v
              for n, v in params.items()}
        src = r if rows is None else int(rows[r])
        want, lp = definition(logits[src], float(uniforms[r]), **at)
        assert got[r].item() == want, f"row {r}: {got[r].item()} for {want}, {at}"
        have = logprob[r].item()
        assert have == lp or abs(have - lp) <= 2.0 ** -24 * abs(lp) + 1e-9, (r, have, lp)
    return got


def logits_of(device, rows, vocab, dtype, seed, spread=1.5):
    gen = torch.Generator().manual_seed(seed)
    x = -(-torch.rand(rows, vocab, generator=gen).clamp_(1e-7, 1 - 1e-7).log()).log() * spread
    return x.to(dtype).to(device)


def uniforms_of(rows, seed):
    return torch.rand(rows, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("vocab", [1, 2, 7, 128, 1000, 2048, 2049, 5003, 32000, 151936])
@pytest.mark.parametrize("params", [
    {}, {"top_k": 40}, {"top_p": 0.9}, {"min_p": 0.05}, {"temperature": 0.7, "top_k": 1500,
                                                        "top_p": 0.95, "min_p": 0.001},
    {"temperature": 1.6, "top_k": 9000, "top_p": 0.999}], ids=str)
def test_definition(device, dtype, vocab, params):
    x = logits_of(device, 5, vocab, dtype, seed=vocab)
    check(x, uniforms_of(5, vocab + 1), **params)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_parameters_of_each_row(device, dtype):
    rows = 24
    gen = torch.Generator().manual_seed(5)
    x = logits_of(device, rows, 20011, dtype, seed=2)
    t = 0.3 + torch.rand(rows, generator=gen)
    t[3] = 0.0
    k = torch.randint(-1, 3000, (rows,), generator=gen)
    k[5], k[6], k[7] = 1, 0, 10 ** 9
    p = torch.rand(rows, generator=gen)
    p[8], p[9], p[10] = 1.0, 0.0, 1.5
    m = 0.2 * torch.rand(rows, generator=gen)
    m[11], m[12], m[13] = 1.0, 2.0, -1.0
    u = uniforms_of(rows, 6)
    check(x, u, temperature=t, top_k=k, top_p=p, min_p=m)
    check(x, u.double(), temperature=t, top_k=k.int(), top_p=0.8, min_p=m)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [100, 2048, 4097, 60001])
@pytest.mark.parametrize("params", [{}, {"top_k": 33}, {"top_k": 3000}, {"top_p": 0.5},
                                    {"min_p": 0.5}], ids=str)
def test_equal_logits(device, dtype, vocab, params):
    """Whole rows of ties: the order is the index's."""
    x = torch.full((4, vocab), -3.25, dtype=dtype, device=device)
    x[1] = 0.0
    x[1, ::2] = -0.0
    # Half the row lies 700 halvings below: no weight at all.
    x[2, vocab // 2:] = -500.0
    # Blocks of equal values, far apart and near.
    x[3] = torch.arange(vocab, device=device).div(vocab / 5).floor().to(dtype) / 8
    check(x, torch.tensor([0.0, 0.37, 0.9999, 0.61]), **params)


def test_crowded_bins(device):
    """More values in one bin than the list holds, some equal, some apart by
    one FP32 step; temperatures that squeeze a row into one bin."""
    gen = torch.Generator().manual_seed(9)
    x = (1.0 + torch.randint(0, 60, (6, 30000), generator=gen) * 2.0 ** -23).to(device)
    x[:, 17] = 8.0
    x[3:] += 1e-3 * torch.randn(3, 30000, generator=gen).to(device)
    u = torch.tensor([0.1, 0.5, 0.999, 0.3, 0.7, 0.95])
    check(x, u)
    check(x, u, top_k=12345, top_p=0.97)
    check(x, u, temperature=50.0, top_p=0.4, min_p=0.1)
    check(x, u, temperature=1e6, top_k=29000)
    check(x, u, temperature=math.inf)
    check(x, u, temperature=1e-6)
    check(x, u, temperature=1e-40)


@pytest.mark.parametrize("vocab", [50, 9000])
def test_masked_infinite_and_missing_values(device, vocab):
    x = logits_of(device, 8, vocab, torch.float32, seed=11)
    x[0] = -math.inf
    x[1, 1:] = -math.inf
    x[2, ::2] = -math.inf
    x[3, ::3] = math.nan
    x[4] = math.nan
    x[5, 20:23] = math.inf
    x[6] = torch.finfo(torch.float32).min
    x[7, 5] = torch.finfo(torch.float32).max
    u = uniforms_of(8, 12)
    for params in ({}, {"top_k": 10}, {"top_p": 0.5}, {"min_p": 0.01}):
        got = check(x, u, **params)
        assert got[0] == -1 and got[4] == -1 and got[1] == 0 and got[5] == 20


def test_uniforms_at_and_past_their_ends(device):
    x = logits_of(device, 6, 3001, torch.float32, seed=13)
    u = torch.tensor([0.0, 1.0, -0.5, 2.0, math.nan, 1 - 2.0 ** -24])
    got = sample_tokens(x, u.to(device)).tolist()
    order = torch.argsort(x.cpu().double(), dim=-1, descending=True, stable=True)
    assert [got[0], got[2], got[4]] == order[[0, 2, 4], 0].tolist()
    # From 1 on: the last of the order that weighs anything (all do here).
    assert got[1] == order[1, -1] and got[3] == order[3, -1]


def test_rows_strides_and_order(device):
    wide = logits_of(device, 9, 4100, torch.bfloat16, seed=14)
    x = wide[:, 3:4003]  # rows start at 2-byte alignment
    u = uniforms_of(5, 15)
    rows = torch.tensor([8, 0, 8, 3, 1])
    check(x, u, rows=rows, top_p=0.9)
    got = sample_tokens(x, u.to(device), rows=torch.tensor([0, -1, 9, 2 ** 40, 8], device=device))
    assert got[1:4].tolist() == [-1, -1, -1] and got[0] >= 0 and got[4] >= 0
    assert sample_tokens(x[:0], u[:0].to(device)).shape == (0,)


def test_same_numbers_same_tokens(device):
    x = logits_of(device, 32, 151936, torch.bfloat16, seed=16)
    u = uniforms_of(32, 17).to(device)
    first = sample_tokens(x, u, top_p=0.95, temperature=1.3)
    for _ in range(3):
        assert torch.equal(first, sample_tokens(x, u, top_p=0.95, temperature=1.3))


def test_captured_and_replayed_on_another_stream(device):
    x = logits_of(device, 7, 50000, torch.float32, seed=18)
    u = uniforms_of(7, 19).to(device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        sample_tokens(x, u, top_p=0.9)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lp = sample_tokens(x, u, top_p=0.9, return_logprobs=True)
    for i in range(3):
        x.copy_(logits_of(device, 7, 50000, torch.float32, seed=20 + i))
        u.copy_(uniforms_of(7, 30 + i))
        graph.replay()
        torch.cuda.synchronize()
        want, want_lp = sample_tokens(x, u, top_p=0.9, return_logprobs=True)
        assert torch.equal(out, want) and torch.equal(lp, want_lp)
