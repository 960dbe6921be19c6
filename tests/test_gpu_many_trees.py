"""Batches of many drafted trees and of many weighed requests against 64 bits: past the
sequences that the kernel of 128 rows cuts, past the units that it cuts and puts in order,
and past one item for every workgroup of the kernel of 16 rows."""

from __future__ import annotations

import random

import pytest
import torch

from mini_llm_runtime_amd.kernels.key_eviction import paged_attention_decode_weighted
from mini_llm_runtime_amd.kernels.tree_attention import paged_attention_tree, tree_ancestors

import selection_oracle as so

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def run_trees(device, dtype, heads, counts, past, check=None):
    """Every tree, or those of `check`, against 64 bits; all of them must be finite."""
    hq, hkv, d = heads
    rng = random.Random(len(counts))
    lens = [p + n for p, n in zip(past, counts)]
    k, v, tables = so.pool(lens, 16, hkv, d, dtype, 1)
    parents = [so.random_parents(n, rng) for n in counts]
    total = sum(counts)
    q = torch.randn(total, hq, d, generator=torch.Generator().manual_seed(2)).to(dtype)
    qsl = torch.tensor([0, *counts]).cumsum(0)
    bits = tree_ancestors(torch.tensor(sum(parents, [])).to(device), qsl.to(device), max(counts))
    out = torch.full((total + 3, hq, d), 7.0, dtype=dtype, device=device)
    got = paged_attention_tree(q.to(device), k.to(device), v.to(device), tables.to(device),
                               qsl.to(device), torch.tensor(lens).to(device), bits, 16,
                               out=out[:total]).cpu()
    assert (out[total:] == 7.0).all() and got.isfinite().all()
    for i in range(len(counts)) if check is None else check:
        n = lens[i]
        if counts[i] == 0:
            continue
        seen = torch.zeros(counts[i], n, dtype=torch.bool)
        seen[:, :past[i]] = True
        for r, path in enumerate(so.paths(parents[i])):
            seen[r, [past[i] + j for j in path]] = True
        slot, rows = so.slots(tables[i], n, 16), slice(int(qsl[i]), int(qsl[i + 1]))
        want, bound, _, _ = so.attend(q[rows], k.view(-1, hkv, d)[slot], v.view(-1, hkv, d)[slot],
                                      seen, d ** -0.5, 0.0, dtype)
        so.assert_within(got[rows], want, bound, f"sequence {i}")


def sizes(seqs, most, past, seed, empty=0.1):
    """Trees of 1 to `most` tokens, some of none, the longest among them."""
    rng = random.Random(seed)
    counts = [0 if rng.random() < empty else rng.randint(1, most) for _ in range(seqs)]
    counts[rng.randrange(seqs)] = most
    before = [rng.randint(0, past) for _ in range(seqs)]
    before[rng.randrange(seqs)] = past
    return counts, before


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("seqs", [511, 512, 513])
def test_sequences_that_are_cut_and_that_are_not(device, dtype, seqs):
    run_trees(device, dtype, (8, 1, 16), *sizes(seqs, 6, 200, seqs))


@pytest.mark.parametrize("heads,seqs", [((32, 8, 16), 150), ((32, 8, 128), 66)])
def test_units_past_four_for_every_slot(device, heads, seqs):
    """Two units of 128 rows a sequence and KV head: left whole, the longest keys first."""
    run_trees(device, BF, heads, *sizes(seqs, 40, 180, seqs))


def test_units_past_those_put_in_order(device):
    """Nine units a sequence for the sake of one large tree."""
    counts, past = sizes(500, 3, 160, 5)
    counts[77] = 40
    run_trees(device, BF, (28, 1, 16), counts, past, check=[*range(60, 100), *range(480, 500)])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("seqs", [257, 600])
def test_short_trees_past_one_item_a_workgroup(device, dtype, seqs):
    """Units of 16 rows left whole, several for a workgroup, some of them without rows."""
    run_trees(device, dtype, (8, 4, 16), *sizes(seqs, 4, 90, seqs))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("most", [100, 700])
def test_weighing_past_one_item_a_workgroup(device, dtype, most):
    """600 requests of 4 KV heads, in one launch (up to 100 keys) and cut into items."""
    rng, hq, hkv, d = random.Random(most), 8, 4, 16
    lens = [0 if rng.random() < 0.1 else rng.randint(1, 100) for _ in range(600)]
    lens[300] = most
    k, v, tables = so.pool(lens, 16, hkv, d, dtype, 1)
    q = torch.randn(600, hq, d, generator=torch.Generator().manual_seed(2)).to(dtype)
    weights = torch.zeros(k.shape[0], hkv, 16, device=device)
    got = paged_attention_decode_weighted(q.to(device), k.to(device), v.to(device), weights,
                                          tables.to(device), torch.tensor(lens).to(device), 16,
                                          validate=False).cpu()
    want = torch.zeros(weights.shape, dtype=torch.float64)
    size = torch.zeros_like(want)
    for i, n in enumerate(lens):
        if n == 0:
            assert (got[i] == 0).all()
            continue
        slot = so.slots(tables[i], n, 16)
        out, bound, p, pb = so.attend(q[i:i + 1], k.view(-1, hkv, d)[slot],
                                      v.view(-1, hkv, d)[slot],
                                      torch.ones(1, n, dtype=torch.bool), d ** -0.5, 0.0, dtype)
        so.assert_within(got[i:i + 1], out, bound, f"request {i}")
        add = p[0].view(hkv, 2, n).sum(1).T
        want[slot // 16, :, slot % 16] = add
        size[slot // 16, :, slot % 16] = pb[0].view(hkv, 2, n).sum(1).T + 3 * 2.0 ** -24 * add
    so.assert_within(weights, want, size, "weights")
