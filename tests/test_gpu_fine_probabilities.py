"""What 16-bit drafted trees, weighing and sparse decodes hold of a probability before it
meets V: 2^-15 of it in bf16 and 2^-21 in fp16, not the 2^-8 and 2^-11 of one rounding to
the type. Scores lie close together here, so that neither they nor the exponentials hide it.

The tolerance, against 64 bits: half a step of the type for the result's own rounding, the
oracle's bound for FP32 scores, exponentials and sums, and for each key the parts' error
times its weight and |v|; in fp16 also 2^-31 times |v|, as parts below 2^-24 may be dropped
from numbers of which the row's largest is at least 2^7.
"""

from __future__ import annotations

import random

import pytest
import torch

from mini_llm_runtime_amd.kernels.key_eviction import paged_attention_decode_weighted
from mini_llm_runtime_amd.kernels.sparse_attention import (paged_attention_decode_sparse,
                                                           update_key_bounds)
from mini_llm_runtime_amd.kernels.tree_attention import paged_attention_tree, tree_ancestors

import selection_oracle as so

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16
HEADS = [(14, 2, 64), (8, 2, 128), (6, 2, 40)]


def compare(got, q, k, v, seen, dtype, what):
    """got, q [n, Hq, D] over keys [N, Hkv, D]; seen [n, N] or [n, Hkv, N]."""
    scale = q.shape[2] ** -0.5
    want, bound, _, _ = so.attend(q, k, v, seen, scale)
    size, _, _, _ = so.attend(q, k, v.abs(), seen, scale)
    info = torch.finfo(dtype)
    parts = 2.0 ** -15 if dtype == BF else 2.0 ** -21
    bound = bound + info.eps / 2 * want.abs().clamp(min=info.tiny) + parts * size
    if dtype == FP:
        bound = bound + 2.0 ** -31 * seen.sum(-1).max() * v.double().abs().max()
    so.assert_within(got, want, bound, what)


def few(n, heads, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    return (0.05 * torch.randn(n, heads[0], heads[2], generator=gen)).to(dtype)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("counts,past", [([2, 1, 4], [0, 9, 30]), ([2], [1500]),
                                         ([40, 31], [3, 20]), ([64], [1000])])
def test_trees(device, dtype, heads, counts, past):
    hq, hkv, d = heads
    rng = random.Random(sum(counts))
    lens = [p + n for p, n in zip(past, counts)]
    k, v, tables = so.pool(lens, 16, hkv, d, dtype, 1)
    q = few(sum(counts), heads, dtype, 2)
    parents = [so.random_parents(n, rng) for n in counts]
    qsl = torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()])
    bits = tree_ancestors(torch.tensor(sum(parents, [])).to(device), qsl.to(device), max(counts))
    got = paged_attention_tree(q.to(device), k.to(device), v.to(device), tables.to(device),
                               qsl.to(device), torch.tensor(lens).to(device), bits, 16)
    for i, n in enumerate(lens):
        seen = torch.zeros(counts[i], n, dtype=torch.bool)
        seen[:, :past[i]] = True
        for r, path in enumerate(so.paths(parents[i])):
            seen[r, [past[i] + j for j in path]] = True
        slot, rows = so.slots(tables[i], n, 16), slice(int(qsl[i]), int(qsl[i + 1]))
        compare(got[rows], q[rows], k.view(-1, hkv, d)[slot], v.view(-1, hkv, d)[slot], seen, dtype,
                f"sequence {i}")


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("lens", [[3, 1, 17, 100], [6, 2000, 9]])
def test_weighing(device, dtype, heads, lens):
    hq, hkv, d = heads
    k, v, tables = so.pool(lens, 16, hkv, d, dtype, 1)
    q = few(len(lens), heads, dtype, 2)
    weights = torch.zeros(k.shape[0], hkv, 16, device=device)
    got = paged_attention_decode_weighted(q.to(device), k.to(device), v.to(device), weights,
                                          tables.to(device), torch.tensor(lens).to(device), 16)
    for i, n in enumerate(lens):
        slot = so.slots(tables[i], n, 16)
        compare(got[i:i + 1], q[i:i + 1], k.view(-1, hkv, d)[slot], v.view(-1, hkv, d)[slot],
                torch.ones(1, n, dtype=torch.bool), dtype, f"request {i}")


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("lens,budget", [([3, 1, 17, 100], 4), ([6, 2000, 300], 100)])
def test_sparse(device, dtype, heads, lens, budget):
    hq, hkv, d = heads
    k, v, tables = so.pool(lens, 16, hkv, d, dtype, 1)
    q = few(len(lens), heads, dtype, 2)
    bounds = torch.zeros(k.shape[0], 2, hkv, d, dtype=dtype, device=device)
    args = [x.to(device) for x in (k, v, tables)]
    ctx = torch.tensor(lens).to(device)
    update_key_bounds(args[0], bounds, args[2], ctx, 16)
    got, blocks = paged_attention_decode_sparse(q.to(device), *args[:2], bounds, args[2], ctx, 16,
                                                budget, return_blocks=True)
    for i, n in enumerate(lens):
        seen = torch.zeros(1, hkv, n, dtype=torch.bool)
        for h in range(hkv):
            for j in blocks[i, h][blocks[i, h] >= 0].tolist():
                seen[0, h, 16 * j:16 * j + 16] = True
        slot = so.slots(tables[i], n, 16)
        compare(got[i:i + 1], q[i:i + 1], k.view(-1, hkv, d)[slot], v.view(-1, hkv, d)[slot], seen,
                dtype, f"request {i}")


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("counts", [[4], [40]])
def test_infinite_values_stay(device, dtype, counts):
    """An infinite V at a key that every row sees is that infinity in each, in a tile that
    is seen whole and in one that is not: neither part of a probability turns it into NaN."""
    n = counts[0] + 200
    k, v, tables = so.pool([n], 16, 2, 64, dtype, 1)
    q = few(counts[0], (14, 2, 64), dtype, 2)
    for at, sign in ((5, 1.0), (150, -1.0)):
        v[tables[0, at // 16], at % 16, :, at % 7::9] = sign * torch.inf
    qsl = torch.tensor([0, counts[0]]).to(device)
    parents = torch.full((counts[0],), -1)
    args = [x.to(device) for x in (q, k, v, tables)]
    bits = tree_ancestors(parents.to(device), qsl, counts[0])
    ctx = torch.tensor([n]).to(device)
    got = paged_attention_tree(*args, qsl, ctx, bits, 16)
    seen = torch.zeros(counts[0], n, dtype=torch.bool)
    seen[:, :200] = True
    seen[torch.arange(counts[0]), 200 + torch.arange(counts[0])] = True
    slot = so.slots(tables[0], n, 16)
    keys = k.view(-1, 2, 64)[slot], v.view(-1, 2, 64)[slot]
    want, bound, _, _ = so.attend(q, *keys, seen, 0.125, 0.0, dtype)
    assert want.isinf().any()
    so.assert_within(got, want, bound)
    weights = torch.zeros(k.shape[0], 2, 16, device=device)
    one = torch.ones(1, n, dtype=torch.bool)
    got = paged_attention_decode_weighted(args[0][:1], *args[1:3], weights, args[3], ctx, 16)
    want, bound, _, _ = so.attend(q[:1], *keys, one, 0.125, 0.0, dtype)
    so.assert_within(got, want, bound)
    bounds = torch.zeros(k.shape[0], 2, 2, 64, dtype=dtype, device=device)
    update_key_bounds(args[1], bounds, args[3], ctx, 16)
    got = paged_attention_decode_sparse(args[0][:1], *args[1:3], bounds, args[3], ctx, 16, 16)
    so.assert_within(got, want, bound)
