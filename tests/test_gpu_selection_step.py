"""Drafted trees, eviction and sparse decode as a program uses them: one after the other over
one cache, captured into graphs, on streams of their own, and far behind in a large pool."""

from __future__ import annotations

import random

import pytest
import torch

from mini_llm_runtime_amd.kernels.key_eviction import (compact_keys, evict_keys,
                                                       paged_attention_decode_weighted)
from mini_llm_runtime_amd.kernels.scored_attention import paged_attention_decode_scored
from mini_llm_runtime_amd.kernels.sparse_attention import (paged_attention_decode_sparse,
                                                           update_key_bounds)
from mini_llm_runtime_amd.kernels.tree_attention import paged_attention_tree, tree_ancestors

import selection_oracle as so

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
HQ, HKV, D, BS = 14, 2, 64, 16


def append(cache, tables, start, rows):
    """Writes rows [B, n, Hkv, D] at positions start[b] + i."""
    at = start[:, None] + torch.arange(rows.shape[1], device=start.device)
    block = torch.gather(tables, 1, at // BS)
    cache[block, at % BS] = rows


@pytest.mark.parametrize("dtype", [BF, F32])
def test_drafted_tokens_step_by_step(device, dtype):
    """Trees are drafted, verified and cut to a path; at the end the cache is that of the
    accepted tokens alone, and decode over it sees just them."""
    rng, gen = random.Random(3), torch.Generator().manual_seed(4)
    lens = [20, 37, 64]
    k, v, tables = so.pool([n + 200 for n in lens], BS, HKV, D, dtype, 1)
    truth = [[x.view(-1, HKV, D)[so.slots(tables[i], n, BS)] for i, n in enumerate(lens)]
             for x in (k, v)]
    k, v, tables = k.to(device), v.to(device), tables.to(device)
    for step in range(4):
        count = rng.choice([5, 12, 24])
        parents = [so.random_parents(count, rng) for _ in lens]
        start = torch.tensor(lens)
        new = [torch.randn(3, count, HKV, D, generator=gen).to(dtype) for _ in range(2)]
        for cache, rows in zip((k, v), new):
            append(cache, tables, start.to(device), rows.to(device))
        qsl = torch.arange(4) * count
        q = torch.randn(3 * count, HQ, D, generator=gen).to(dtype)
        bits = tree_ancestors(torch.tensor(sum(parents, [])).to(device), qsl.to(device), count)
        got = paged_attention_tree(q.to(device), k, v, tables, qsl.to(device),
                                   (start + count).to(device), bits, BS)
        paths = [so.paths(p) for p in parents]
        kept = torch.full((3, count), -1)
        for i, n in enumerate(lens):
            keys = [torch.cat([truth[x][i], new[x][i]]) for x in range(2)]
            seen = torch.zeros(count, n + count, dtype=torch.bool)
            seen[:, :n] = True
            for r, s in enumerate(paths[i]):
                seen[r, [n + j for j in s]] = True
            want, bound, _, _ = so.attend(q[i * count:(i + 1) * count], *keys, seen, D ** -0.5,
                                          0.0, dtype)
            so.assert_within(got[i * count:(i + 1) * count], want, bound, f"step {step}")
            path = sorted(rng.choice(paths[i]))
            kept[i, :len(path)] = torch.tensor(path) + n
            for x in range(2):
                truth[x][i] = torch.cat([truth[x][i], new[x][i][path]])
        compact_keys(k, v, tables, kept.to(device), BS, start=start.to(device))
        lens = [len(t) for t in truth[0]]
    q = torch.randn(3, HQ, D, generator=gen).to(dtype)
    got = paged_attention_decode_scored(q.to(device), k, v, tables, torch.tensor(lens).to(device),
                                        BS)
    for i, n in enumerate(lens):
        want, bound, _, _ = so.attend(q[i:i + 1], truth[0][i], truth[1][i],
                                      torch.ones(1, n, dtype=torch.bool), D ** -0.5, 0.0, dtype)
        so.assert_within(got[i:i + 1], want, bound)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_cache_that_is_cut_as_it_grows(device, dtype):
    """Weighing steps, and a cut whenever a request passes its budget: every KV head keeps
    keys of its own, which later steps see alone."""
    gen = torch.Generator().manual_seed(4)
    lens, budget = [30, 44], 40
    k, v, tables = so.pool([64, 64], BS, HKV, D, dtype, 1)
    weights = torch.zeros(k.shape[0], HKV, BS)
    # Of each request and KV head: keys, values, sums.
    truth = [[[x.view(-1, HKV, D)[so.slots(tables[i], n, BS), h] for x in (k, v)] +
              [torch.zeros(n, dtype=torch.float64)] for h in range(HKV)]
             for i, n in enumerate(lens)]
    k, v, tables, weights = (x.to(device) for x in (k, v, tables, weights))
    for step in range(12):
        start = torch.tensor(lens)
        new = [torch.randn(2, 1, HKV, D, generator=gen).to(dtype) for _ in range(2)]
        for cache, rows in zip((k, v), new):
            append(cache, tables, start.to(device), rows.to(device))
        lens = [n + 1 for n in lens]
        ctx = torch.tensor(lens).to(device)
        q = torch.randn(2, HQ, D, generator=gen).to(dtype)
        got = paged_attention_decode_weighted(q.to(device), k, v, weights, tables, ctx, BS)
        group = HQ // HKV
        for i, n in enumerate(lens):
            for h in range(HKV):
                t = truth[i][h]
                for x in range(2):
                    t[x] = torch.cat([t[x], new[x][i, :, h]])
                want, bound, p, _ = so.attend(
                    q[i:i + 1, h * group:(h + 1) * group], t[0][:, None], t[1][:, None],
                    torch.ones(1, n, dtype=torch.bool), D ** -0.5, 0.0, dtype)
                so.assert_within(got[i:i + 1, h * group:(h + 1) * group], want, bound, f"{step}")
                t[2] = torch.cat([t[2], torch.zeros(1, dtype=torch.float64)]) + p[0].sum(0)
        if step % 4 == 3:
            kept, new_lens = evict_keys(k, v, weights, tables, ctx, BS, budget, sinks=2, recent=8)
            for i, n in enumerate(lens):
                for h in range(HKV):
                    stay = [j for j in kept[i, h].tolist() if j >= 0]
                    # The sums are close, so the choice is that of the exact ones but for ties
                    # within their error.
                    t = truth[i][h]
                    want = so.choose(t[2], 2, 8, budget)
                    if n > budget:
                        left = sorted(set(want) - set(stay)) + sorted(set(stay) - set(want))
                        assert all(abs(t[2][a] - t[2][b]) < 1e-3 for a in left for b in left)
                    else:
                        assert stay == want
                    truth[i][h] = [x[stay] for x in t]
            lens = new_lens.tolist()
            assert lens == [min(n, budget) for n in ctx.tolist()]


@pytest.mark.parametrize("dtype", [BF, F32])
def test_bounds_that_follow_a_growing_cache(device, dtype):
    """Bounds brought up to date step by step are those of a whole pass, and sparse decode
    chooses by them."""
    gen = torch.Generator().manual_seed(4)
    lens = [100, 333]
    k, v, tables = so.pool([200, 400], BS, HKV, D, dtype, 1)
    k, v, tables = k.to(device), v.to(device), tables.to(device)
    bounds = torch.zeros(k.shape[0], 2, HKV, D, dtype=dtype, device=device)
    update_key_bounds(k, bounds, tables, torch.tensor(lens).to(device), BS)
    for count in (1, 1, 20, 3, 16):
        start = torch.tensor(lens).to(device)
        for cache in (k, v):
            append(cache, tables, start,
                   torch.randn(2, count, HKV, D, generator=gen).to(dtype).to(device))
        lens = [n + count for n in lens]
        ctx = torch.tensor(lens).to(device)
        update_key_bounds(k, bounds, tables, ctx, BS, starts=start, max_new=count)
        q = torch.randn(2, HQ, D, generator=gen).to(dtype)
        got, blocks = paged_attention_decode_sparse(q.to(device), k, v, bounds, tables, ctx, BS, 5,
                                                    recent=2, return_blocks=True)
        for i, n in enumerate(lens):
            table, keys = tables[i].cpu(), k.cpu()
            low = torch.stack([keys[table[j], :min(BS, n - j * BS)].amin(0)
                               for j in range(-(-n // BS))])
            high = torch.stack([keys[table[j], :min(BS, n - j * BS)].amax(0)
                                for j in range(-(-n // BS))])
            score = so.block_scores(q[i], low, high)
            seen = torch.zeros(1, HKV, n, dtype=torch.bool)
            for h in range(HKV):
                stay = so.choose(score[h], 1, 2, 5)
                assert blocks[i, h].tolist() == stay
                for j in stay:
                    seen[0, h, j * BS:(j + 1) * BS] = True
            slot = so.slots(table, n, BS)
            want, bound, _, _ = so.attend(q[i:i + 1], keys.view(-1, HKV, D)[slot],
                                          v.cpu().view(-1, HKV, D)[slot], seen, D ** -0.5, 0.0,
                                          dtype)
            so.assert_within(got[i:i + 1], want, bound)


class Calls:
    """One of each call over a cache, as a function of static tensors."""

    def __init__(self, device, dtype, lens, seed, far=0):
        gen = torch.Generator().manual_seed(seed)
        k, v, tables = so.pool(lens, BS, HKV, D, dtype, seed)
        self.k, self.v, self.tables = k.to(device), v.to(device), tables.to(device)
        self.lens = torch.tensor(lens).to(device)
        self.weights = torch.rand(k.shape[0], HKV, BS, generator=gen).to(device)
        self.bounds = torch.zeros(k.shape[0], 2, HKV, D, dtype=dtype, device=device)
        self.q = torch.randn(len(lens), HQ, D, generator=gen).to(dtype).to(device)
        nodes = 9
        self.nodes = nodes
        self.qsl = torch.arange(len(lens) + 1).to(device) * nodes
        self.tree_q = torch.randn(len(lens) * nodes, HQ, D, generator=gen).to(dtype).to(device)
        self.parents = torch.tensor(
            sum((so.random_parents(nodes, random.Random(seed + i)) for i in range(len(lens))),
                [])).to(device)
        self.kept = torch.tensor([[n - 5, n - 3, n - 2] for n in lens]).to(device)
        self.start = self.lens - 6

    def __call__(self):
        """Leaves the cache as it was, but for the sums and the last rows."""
        bits = tree_ancestors(self.parents, self.qsl, self.nodes)
        tree = paged_attention_tree(self.tree_q, self.k, self.v, self.tables, self.qsl, self.lens,
                                    bits, BS, max_query_len=self.nodes, validate=False)
        out = paged_attention_decode_weighted(self.q, self.k, self.v, self.weights, self.tables,
                                              self.lens, BS, validate=False)
        update_key_bounds(self.k, self.bounds, self.tables, self.lens, BS, validate=False)
        sparse, blocks = paged_attention_decode_sparse(
            self.q, self.k, self.v, self.bounds, self.tables, self.lens, BS, 4, recent=2,
            return_blocks=True, validate=False)
        compact_keys(self.k, self.v, self.tables, self.kept, BS, start=self.start, validate=False)
        kept, lens = evict_keys(self.k, self.v, self.weights, self.tables, self.lens, BS, 60,
                                sinks=2, recent=10, validate=False)
        return tree, out, sparse, blocks, kept, lens

    def state(self):
        return [x.clone() for x in (self.k, self.v, self.weights, self.bounds)]

    def restore(self, state):
        for x, y in zip((self.k, self.v, self.weights, self.bounds), state):
            x.copy_(y)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_captured_and_replayed(device, dtype):
    """Two graphs of the same calls over caches of their own, replayed in turn with eager
    work and synchronizations in between, give what eager calls give, every time."""
    calls = [Calls(device, dtype, lens, seed) for seed, lens in
             enumerate(([70, 500, 6], [3000, 90]))]
    graphs, captured, states, eager = [], [], [], []
    for c in calls:
        states.append(c.state())
        eager.append([x.clone() for x in c()] + c.state())
        c.restore(states[-1])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured.append(c())
        graphs.append(graph)
    for turn in range(4):
        for c, graph, got, state, want in zip(calls, graphs, captured, states, eager):
            c.restore(state)
            graph.replay()
            junk = torch.randn(1 << 20, device=device).sort()  # eager work of the program's own
            if turn % 2:
                torch.cuda.synchronize()
            for x, y in zip([*got, *c.state()], want):
                assert torch.equal(x, y)
            del junk
            c.restore(state)
            for x, y in zip([*c(), *c.state()], want):
                assert torch.equal(x, y)


def test_two_streams_at_once(device):
    """Calls on two streams share nothing."""
    calls = [Calls(device, BF, lens, seed) for seed, lens in enumerate(([700, 500, 60], [3000, 90]))]
    states = [c.state() for c in calls]
    want = []
    for c, state in zip(calls, states):
        want.append([x.clone() for x in c()] + c.state())
        c.restore(state)
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for c, stream, state in zip(calls, streams, states):
            with torch.cuda.stream(stream):
                c.restore(state)
                got.append([*c(), *c.state()])
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            for x, y in zip(a, b):
                assert torch.equal(x, y)


def test_far_behind_in_a_large_pool(device):
    """Blocks whose elements and bytes lie past 32 bits."""
    hkv, d, blocks = 8, 128, 140_000  # 4.6 GB a cache
    lens = [100, 70]
    small_k, small_v, tables = so.pool(lens, BS, hkv, d, BF, 3)
    far = tables + (blocks - small_k.shape[0])
    far[tables < 0] = -1
    gen = torch.Generator().manual_seed(1)
    q = torch.randn(2, 32, d, generator=gen).to(BF).to(device)
    tree_q = torch.randn(8, 32, d, generator=gen).to(BF).to(device)
    weights = torch.rand(small_k.shape[0], hkv, BS, generator=gen)
    ctx = torch.tensor(lens).to(device)
    results = []
    for table, first in ((tables, 0), (far, blocks - small_k.shape[0])):
        total = small_k.shape[0] + first
        k = torch.empty(total, BS, hkv, d, dtype=BF, device=device)
        v = torch.empty_like(k)
        w = torch.empty(total, hkv, BS, device=device)
        bounds = torch.empty(total, 2, hkv, d, dtype=BF, device=device)
        k[first:], v[first:], w[first:] = small_k.to(device), small_v.to(device), weights.to(device)
        t = table.to(device)
        bounds[first:] = 0
        bits = torch.full((8, 1), 15, device=device)
        out = [paged_attention_tree(tree_q, k, v, t, torch.tensor([0, 4, 8]).to(device), ctx, bits,
                                    BS),
               paged_attention_decode_weighted(q, k, v, w, t, ctx, BS)]
        update_key_bounds(k, bounds, t, ctx, BS)
        out += paged_attention_decode_sparse(q, k, v, bounds, t, ctx, BS, 4, return_blocks=True)
        out += evict_keys(k, v, w, t, ctx, BS, 50, sinks=2, recent=10)
        out += [x[first:].clone() for x in (k, v, w, bounds)]
        results.append(out)
        del k, v, w, bounds
        torch.cuda.empty_cache()
    for x, y in zip(*results):
        assert torch.equal(x, y)
