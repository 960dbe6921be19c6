"""Drafted trees, key eviction and sparse decode in 64 bits on the CPU, with bounds on what
FP32 arithmetic and 16-bit operands may change. The bounds of attention are those of
scored_oracle.py, for any set of visible keys; a weight, which is not rounded to 16 bits, is
off by twice the largest error of a score, and by 2^-18 of itself for exponentials and sums.
"""

from __future__ import annotations

import random

import torch


def attend(q, k, v, seen, scale, cap=0.0, dtype=torch.float32):
    """q [n, Hq, D] over keys [N, Hkv, D] where seen [n, N] or [n, Hkv, N]: out and its
    bound [n, Hq, D], weights and theirs [n, Hq, N], all in 64 bits."""
    n, hq, d = q.shape
    hkv = k.shape[1]
    q, k, v = q.double(), k.double(), v.double()
    if seen.ndim == 2:
        seen = seen[:, None].expand(-1, hkv, -1)
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    weights = torch.zeros(n, hq, k.shape[0], dtype=torch.float64)
    weight_bound = torch.zeros_like(weights)
    half = torch.finfo(dtype).eps / 2
    if k.shape[0] == 0:
        return out, bound, weights, weight_bound
    for h in range(hq):
        g = h * hkv // hq
        visible = seen[:, g]
        used = visible.any(0)[:, None]
        # What is hidden may hold anything: it takes no part, not even times 0.
        kh, vh = torch.where(used, k[:, g], 0.0), torch.where(used, v[:, g], 0.0)
        x = q[:, h] @ kh.T * scale
        terms = q[:, h].abs() @ kh.abs().T
        # Finite terms that together pass the largest 32-bit number may end as infinity or
        # NaN whatever their order, and the row with them: no bound holds it.
        over = ((terms > torch.finfo(torch.float32).max) & terms.isfinite()
                & visible).any(-1, keepdim=True)
        err = (d + 2) * 2.0 ** -24 * abs(scale) * terms
        if cap:
            x = cap * torch.tanh(x / cap)
            err = err + 2.0 ** -21 * cap
        err = err + 2.0 ** -21 * x.abs()
        x = x.masked_fill(~visible, -torch.inf)
        empty = ~visible.any(-1)
        w = torch.where(visible, (x - x.amax(-1, keepdim=True)).exp(), 0.0)
        l = w.sum(-1, keepdim=True)
        p = torch.where(empty[:, None], 0.0, w / l)
        worst = err.masked_fill(~visible, 0.0).amax(-1, keepdim=True)
        rel = 2 * worst + 2.0 ** -18
        weights[:, h], weight_bound[:, h] = p, rel * p + 1e-37
        rel = rel + (half if dtype != torch.float32 else 0.0)
        clean = torch.where(vh.isfinite(), vh, 0.0)
        o, size = p @ clean, p @ clean.abs()
        extra = 0.0
        if dtype == torch.float16:
            extra = 2.0 ** -25 * (visible.double() @ clean.abs()) / l.clamp(min=1.0)
        # Rows that see a V that is not finite: NaN or infinite there.
        for j in (~vh.isfinite()).any(-1).nonzero().flatten().tolist():
            rows = visible[:, j].nonzero().flatten()
            o[rows] = o[rows] + p[rows, j, None] * torch.where(vh[j].isfinite(), 0.0, vh[j])
        out[:, h] = o
        tiny = torch.finfo(dtype).tiny
        bound[:, h] = torch.where(empty[:, None], 0.0,
                                  half * o.abs().clamp(min=tiny) + rel * size + extra)
        bound[:, h].masked_fill_(over, torch.inf)
        weight_bound[:, h].masked_fill_(over, torch.inf)
    return out, bound, weights, weight_bound


def choose(score, sinks, recent, budget):
    """The places of score [n] that stay, ascending."""
    n = len(score)
    if n <= budget:
        return list(range(n))
    value = [float("-inf") if s != s else s for s in score.tolist()]
    middle = sorted(range(sinks, n - recent), key=lambda i: (-value[i], i))
    return sorted([*range(sinks), *middle[:budget - sinks - recent], *range(n - recent, n)])


def block_scores(q, low, high):
    """q [Hq, D], bounds [n, Hkv, D] in 64 bits: [Hkv, n]."""
    n, hkv, d = low.shape
    group = q.shape[0] // hkv
    out = torch.full((hkv, n), -torch.inf, dtype=torch.float64)
    for h in range(q.shape[0]):
        g, x = h // group, q[h].double()
        s = torch.where(x >= 0, x * high[:, g].double(), x * low[:, g].double()).sum(-1)
        out[g] = torch.maximum(out[g], torch.where(s.isnan(), -torch.inf, s))
    return out


def paths(parents):
    """For each node of one tree the set of itself and its ancestors."""
    out = []
    for i in range(len(parents)):
        seen, at = set(), i
        while 0 <= at < len(parents) and at not in seen:
            seen.add(at)
            at = parents[at]
        out.append(seen)
    return out


def random_parents(n, rng):
    return [-1 if i == 0 or rng.random() < 0.1 else rng.randrange(i) for i in range(n)]


def pool(lens, block_size, hkv, d, dtype, seed, spare=2, device="cpu", width=None):
    """A cache with shuffled tables for these lengths: k, v, tables (-1 past their ends)."""
    gen = torch.Generator().manual_seed(seed)
    need = [-(-n // block_size) for n in lens]
    blocks = sum(need) + spare
    perm = list(range(blocks))
    random.Random(seed).shuffle(perm)
    k = torch.randn(blocks, block_size, hkv, d, generator=gen).to(dtype)
    v = torch.randn(blocks, block_size, hkv, d, generator=gen).to(dtype)
    tables = torch.full((len(lens), max(need + [1]) if width is None else width), -1)
    at = 0
    for i, n in enumerate(need):
        tables[i, :n] = torch.tensor(perm[at:at + n])
        at += n
    return k, v, tables


def slots(table, count, block_size, first=0):
    at = torch.arange(first, count)
    return table[at // block_size] * block_size + at % block_size


def assert_within(got, want, bound, what=""):
    got = got.double().cpu()
    same = (got == want) | (got.isnan() & want.isnan())
    bad = ~same & ~((got - want).abs() <= bound) & ~torch.as_tensor(bound == torch.inf)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} past the bound, first at "
                           f"{bad.nonzero()[0].tolist()}: {got[bad][0]} for {want[bad][0]}, "
                           f"bound {bound.expand_as(got)[bad][0]}")
