"""Weighing decode, eviction and compaction against 64 bits and exact copies."""

from __future__ import annotations

import random

import pytest
import torch

from mini_llm_runtime_amd.kernels.key_eviction import (compact_keys, evict_keys,
                                                       paged_attention_decode_weighted)
from mini_llm_runtime_amd.kernels.scored_attention import paged_attention_decode_scored

import selection_oracle as so

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def weigh(device, dtype, heads, lens, block_size=16, cap=0.0, seed=0, validate=True, change=None):
    hq, hkv, d = heads
    k, v, tables = so.pool(lens, block_size, hkv, d, dtype, seed)
    gen = torch.Generator().manual_seed(seed + 1)
    q = torch.randn(len(lens), hq, d, generator=gen).to(dtype)
    weights = torch.rand(k.shape[0], hkv, block_size, generator=gen)
    if change is not None:
        change(q, k, v, tables)
    total = weights.to(device)
    got = paged_attention_decode_weighted(
        q.to(device), k.to(device), v.to(device), total, tables.to(device),
        torch.tensor(lens).to(device), block_size, softcap=cap, validate=validate)
    want_w, bound_w = weights.double(), torch.zeros(weights.shape, dtype=torch.float64)
    for i, n in enumerate(lens):
        slot = so.slots(tables[i], n, block_size)
        seen = torch.ones(1, n, dtype=torch.bool)
        want, bound, p, pb = so.attend(q[i:i + 1], k.view(-1, hkv, d)[slot],
                                       v.view(-1, hkv, d)[slot], seen, d ** -0.5, cap, dtype)
        so.assert_within(got[i:i + 1], want, bound, f"request {i}")
        if n == 0:
            continue
        block, at = slot // block_size, slot % block_size
        add = p[0].view(hkv, hq // hkv, n).sum(1).T
        # FP32 sums of at most `group` weights, and one sum with what was there.
        size = pb[0].view(hkv, hq // hkv, n).sum(1).T + (hq // hkv + 1) * 2.0 ** -24 * add
        want_w[block[-1], :, at[-1]] = 0
        want_w[block, :, at] += add
        bound_w[block, :, at] = size + 2.0 ** -24 * want_w[block, :, at]
    so.assert_within(total, want_w, bound_w, "weights")
    return got, total


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("heads", [(14, 2, 64), (8, 2, 128), (4, 4, 96), (6, 2, 40), (40, 2, 16)])
def test_weighing(device, dtype, heads):
    weigh(device, dtype, heads, [1, 2, 16, 17, 100, 300])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("block_size", [1, 5, 8, 32, 24])
def test_weighing_block_sizes(device, dtype, block_size):
    weigh(device, dtype, (4, 2, 64), [1, 31, 130], block_size=block_size)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("lens", [[1], [1023], [1024], [1025], [5000, 3], [128] * 40])
def test_weighing_lengths(device, dtype, lens):
    weigh(device, dtype, (14, 2, 64), lens)


@pytest.mark.parametrize("dtype", [BF, FP, F32])
def test_weighing_capped(device, dtype):
    weigh(device, dtype, (14, 2, 64), [40, 200], cap=10.0)


def test_weighing_many_heads_of_a_group(device):
    weigh(device, BF, (80, 1, 32), [1, 77, 400])


def test_weighing_padded_rows(device):
    """Lengths of 0: zeros, and no weight changes."""
    got, _ = weigh(device, BF, (14, 2, 64), [0, 40, 0], validate=False)
    assert (got[0] == 0).all() and (got[2] == 0).all()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_weighing_with_odd_values(device, dtype):
    """What lies behind a request's end is not read; a V that is not finite does not touch
    the weights."""
    def change(q, k, v, tables):
        k[tables[0, 2], 8:] = float("nan")
        v[tables[0, 2], 8:] = float("nan")
        v[tables[1, 0], 3] = float("inf")

    weigh(device, dtype, (14, 2, 64), [40, 30], change=change)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_weighing_is_the_scored_decode(device, dtype):
    k, v, tables = so.pool([1000, 30], 16, 2, 64, dtype, 5)
    q = torch.randn(2, 14, 64, generator=torch.Generator().manual_seed(1)).to(dtype)
    args = [x.to(device) for x in (q, k, v)]
    lens = torch.tensor([1000, 30]).to(device)
    tables = tables.to(device)
    first = None
    for _ in range(3):  # the same every time, bit for bit
        weights = torch.zeros(k.shape[0], 2, 16, device=device)
        got = paged_attention_decode_weighted(*args, weights, tables, lens, 16)
        first = weights if first is None else first
        assert torch.equal(first, weights)
    torch.testing.assert_close(got, paged_attention_decode_scored(*args, tables, lens, 16),
                               rtol=0, atol=2.0 ** -7 if dtype == BF else 1e-5)
    # A request's weights sum to its heads.
    total = [weights[tables[i][tables[i] >= 0]].sum().item() for i in range(2)]
    assert abs(total[0] - 14) < 1e-3 and abs(total[1] - 14) < 1e-3


def test_weighing_shared_blocks(device):
    """Two requests over the same first blocks: both add to their keys."""
    k, v, tables = so.pool([64, 80], 16, 2, 64, F32, 5)
    tables[1, :3] = tables[0, :3]
    q = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(1))
    weights = torch.zeros(k.shape[0], 2, 16, device=device)
    paged_attention_decode_weighted(q.to(device), k.to(device), v.to(device), weights,
                                    tables.to(device), torch.tensor([64, 80]).to(device), 16)
    want = torch.zeros(weights.shape, dtype=torch.float64)
    for i, n in enumerate((64, 80)):
        slot = so.slots(tables[i], n, 16)
        _, _, p, _ = so.attend(q[i:i + 1], k.view(-1, 2, 64)[slot], v.view(-1, 2, 64)[slot],
                               torch.ones(1, n, dtype=torch.bool), 0.125)
        want[slot // 16, :, slot % 16] += p[0].view(2, 2, n).sum(1).T
    so.assert_within(weights, want, torch.full_like(want, 1e-5))


def cut(device, dtype, heads, lens, budget, sinks, recent, weights=None, block_size=16, seed=0,
        validate=True, width=None):
    hkv, d = heads
    k, v, tables = so.pool(lens, block_size, hkv, d, dtype, seed, width=width)
    gen = torch.Generator().manual_seed(seed + 1)
    w = torch.rand(k.shape[0], hkv, block_size, generator=gen)
    if weights is not None:
        weights(w, tables)
    want = [x.clone() for x in (k, v, w)]
    kept_want = torch.full((len(lens), hkv, budget), -1)
    for i, n in enumerate(lens):
        slot = so.slots(tables[i], n, block_size)
        for h in range(hkv):
            stay = so.choose(w[slot // block_size, h, slot % block_size], sinks, recent, budget)
            kept_want[i, h, :len(stay)] = torch.tensor(stay, dtype=torch.long)
            src, dst = slot[stay], slot[:len(stay)]
            for x, y in zip(want[:2], (k, v)):
                x.view(-1, hkv, d)[dst, h] = y.view(-1, hkv, d)[src, h]
            want[2][dst // block_size, h, dst % block_size] = (
                w[src // block_size, h, src % block_size])
    k, v, w = (x.to(device) for x in (k, v, w))
    kept, new_lens = evict_keys(k, v, w, tables.to(device), torch.tensor(lens).to(device),
                                block_size, budget, sinks=sinks, recent=recent, validate=validate)
    assert torch.equal(kept.cpu(), kept_want)
    assert new_lens.tolist() == [min(n, budget) for n in lens]
    for got, x in zip((k, v, w), want):  # bit for bit, NaN too
        bits = torch.int32 if x.element_size() == 4 else torch.int16
        assert torch.equal(got.cpu().view(bits), x.view(bits))


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("heads", [(2, 64), (1, 128), (3, 8), (4, 80), (2, 256)])
def test_eviction(device, dtype, heads):
    cut(device, dtype, heads, [1, 40, 41, 64, 300], 40, 4, 10)


@pytest.mark.parametrize("budget,sinks,recent", [
    (0, 0, 0), (1, 0, 0), (1, 1, 0), (1, 0, 1), (10, 10, 0), (10, 0, 10), (10, 4, 6), (64, 0, 0), (65, 1, 1)])
def test_eviction_budgets(device, budget, sinks, recent):
    cut(device, BF, (2, 64), [1, 9, 10, 11, 66, 200], budget, sinks, recent)


@pytest.mark.parametrize("lens,budget", [([20000, 9000], 7000), ([40000], 1000), ([16384], 16383),
                                         ([1025, 1030], 1024)])
def test_long_eviction(device, lens, budget):
    cut(device, F32, (2, 8), lens, budget, 4, budget // 4)


@pytest.mark.parametrize("block_size", [1, 5, 24, 64])
def test_eviction_block_sizes(device, block_size):
    cut(device, BF, (2, 64), [30, 77, 150], 33, 2, 8, block_size=block_size)


@pytest.mark.parametrize("kind", ["equal", "two values", "nan", "infinite", "zeros", "negative",
                                  "neighbours"])
def test_eviction_by_odd_weights(device, kind):
    """Ties go to the lower position, NaN counts as -infinity, -0 as 0."""
    def change(w, tables):
        gen = torch.Generator().manual_seed(9)
        if kind == "equal":
            w.fill_(0.5)
        elif kind == "two values":
            w.copy_((w > 0.7).float())
        elif kind == "nan":
            w[torch.rand(w.shape, generator=gen) < 0.7] = float("nan")
        elif kind == "infinite":
            w[torch.rand(w.shape, generator=gen) < 0.2] = float("inf")
            w[torch.rand(w.shape, generator=gen) < 0.6] = -float("inf")
        elif kind == "zeros":
            w.copy_(torch.where(w < 0.5, 0.0, -0.0))
        elif kind == "negative":
            w.copy_(w - 0.8)
        else:
            w.copy_(1 + (w * 40).floor() * 2.0 ** -23)

    cut(device, BF, (2, 64), [50, 300, 2000], 100, 4, 20, weights=change)


def test_eviction_wide_tables(device):
    cut(device, BF, (2, 64), [50, 300], 100, 4, 20, width=64)


def test_eviction_padded_rows(device):
    cut(device, BF, (2, 64), [0, 120, 0], 33, 4, 20, validate=False)


def moved(k, v, w, tables, kept, start, bs):
    hkv, d = k.shape[2:]
    out = [k.clone(), v.clone(), None if w is None else w.clone()]
    for i in range(len(kept)):
        for h in range(hkv):
            stay = kept[i] if kept.ndim == 2 else kept[i, h]
            stay = stay[stay >= 0]
            to = start[i] + torch.arange(len(stay))
            src = tables[i][stay // bs] * bs + stay % bs
            dst = tables[i][to // bs] * bs + to % bs
            for x, y in zip(out[:2], (k, v)):
                x.view(-1, hkv, d)[dst, h] = y.view(-1, hkv, d)[src, h]
            if w is not None:
                out[2][dst // bs, h, dst % bs] = w[src // bs, h, src % bs]
    return out


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("per_head", [False, True])
@pytest.mark.parametrize("weighted", [False, True])
def test_compaction(device, dtype, per_head, weighted):
    """Lists from none to all of what follows a start, their ends apart."""
    rng = random.Random(4)
    lens, starts, hkv, d = [20, 300, 33, 700, 64], [3, 100, 0, 17, 64], 3, 72
    k, v, tables = so.pool(lens, 16, hkv, d, dtype, 3)
    w = torch.rand(k.shape[0], hkv, 16) if weighted else None
    kept = torch.full((5, hkv, 650), -1)
    for i in range(5):
        for h in range(hkv):
            span = range(starts[i], lens[i])
            stay = sorted(rng.sample(span, int(len(span) * rng.choice([0, 0.1, 0.5, 0.9, 1]))))
            kept[i, h, :len(stay)] = torch.tensor(stay, dtype=torch.long)
    if not per_head:
        kept = kept[:, 1].contiguous()
    want = moved(k, v, w, tables, kept, starts, 16)
    k, v = k.to(device), v.to(device)
    w = None if w is None else w.to(device)
    assert compact_keys(k, v, tables.to(device), kept.to(device), 16,
                        start=torch.tensor(starts).to(device), key_weights=w) is None
    assert torch.equal(k.cpu(), want[0]) and torch.equal(v.cpu(), want[1])
    if weighted:
        assert torch.equal(w.cpu(), want[2])


@pytest.mark.parametrize("drop", [[0], [1], [5], [100], [0, 1, 2, 3], list(range(0, 4000, 2)),
                                  list(range(1, 4000, 777))])
def test_compaction_of_long_rows_by_small_steps(device, drop):
    """Neighbouring rows move by one place: each is read before it is written."""
    n = 4000
    k, v, tables = so.pool([n], 16, 2, 64, BF, 3)
    kept = torch.tensor([[i for i in range(n) if i not in set(drop)]])
    want = moved(k, v, None, tables, kept, [0], 16)
    k, v = k.to(device), v.to(device)
    compact_keys(k, v, tables.to(device), kept.to(device), 16)
    assert torch.equal(k.cpu(), want[0]) and torch.equal(v.cpu(), want[1])


@pytest.mark.parametrize("block_size,n", [(1, 6000), (2, 9001), (48, 6000)])
@pytest.mark.parametrize("hkv,d", [(1, 8), (5, 64)])
def test_compaction_of_wide_tables(device, block_size, n, hkv, d):
    """More blocks than a workgroup holds ids of, one list and several at a time."""
    rng = random.Random(n)
    k, v, tables = so.pool([n, 40], block_size, hkv, d, BF, 3)
    kept = torch.full((2, n), -1)
    for i, count in enumerate((n, 40)):
        stay = sorted(rng.sample(range(count), count * 2 // 3))
        kept[i, :len(stay)] = torch.tensor(stay)
    want = moved(k, v, None, tables, kept, [0, 0], block_size)
    k, v = k.to(device), v.to(device)
    compact_keys(k, v, tables.to(device), kept.to(device), block_size)
    assert torch.equal(k.cpu(), want[0]) and torch.equal(v.cpu(), want[1])


def test_compaction_of_an_accepted_path_behind_a_shared_prefix(device):
    """Requests may share blocks before the start."""
    k, v, tables = so.pool([70, 70], 16, 2, 64, BF, 3)
    tables[1, :3] = tables[0, :3]
    kept = torch.tensor([[50, 53, 60], [49, -1, -1]])
    want = moved(k, v, None, tables, kept, [50, 49], 16)
    k, v = k.to(device), v.to(device)
    compact_keys(k, v, tables.to(device), kept.to(device), 16,
                 start=torch.tensor([50, 49]).to(device))
    assert torch.equal(k.cpu(), want[0]) and torch.equal(v.cpu(), want[1])


def test_compaction_with_bad_blocks(device):
    """With validate=False positions past the table, below 0 and of blocks out of range move
    nothing."""
    k, v, tables = so.pool([64], 16, 2, 64, BF, 3)
    want = [k.clone(), v.clone()]
    flat = [x.view(-1, 2, 64) for x in want]
    src, dst = tables[0, 1] * 16 + 4, tables[0, 0] * 16 + 1
    for x in flat:
        x[dst] = x[src].clone()
    tables[0, 2] = 1 << 40
    kept = torch.tensor([[0, 20, 40, 1000, 1 << 50, -7]])
    k, v = k.to(device), v.to(device)
    compact_keys(k, v, tables.to(device), kept.to(device), 16, validate=False)
    assert torch.equal(k.cpu(), want[0]) and torch.equal(v.cpu(), want[1])


def test_weighing_refuses_a_newest_key_of_two_requests(device):
    """Its entry would be set by one and added to by the other. What is shared and is no
    request's newest key is fine."""
    k, v, tables = so.pool([40, 40], 16, 2, 64, BF, 1)
    q = torch.zeros(2, 4, 64, dtype=BF, device=device)
    weights = torch.zeros(k.shape[0], 2, 16, device=device)
    lens = torch.tensor([40, 40]).to(device)
    for shared, fits in ((2, True), (3, False)):
        tables[1, :shared] = tables[0, :shared]
        args = (q, k.to(device), v.to(device), weights, tables.to(device), lens, 16)
        if fits:
            paged_attention_decode_weighted(*args)
            continue
        before = weights.clone()
        with pytest.raises(ValueError, match="newest key"):
            paged_attention_decode_weighted(*args)
        assert torch.equal(weights, before)


@pytest.mark.parametrize("budget,recent", [(4, 0), (5, 1), (6, 2), (7, 3), (8, 4), (9, 4), (33, 16)])
def test_eviction_with_as_many_recent_keys_as_fit(device, budget, recent):
    """Without `recent`: half the budget, or what the sinks leave of a small one."""
    k, v, tables = so.pool([5, 70], 16, 2, 64, F32, 1)
    w = torch.rand(k.shape[0], 2, 16, generator=torch.Generator().manual_seed(2))
    lens = torch.tensor([5, 70]).to(device)
    results = []
    for more in (dict(recent=recent), dict()):
        own = [x.to(device, copy=True) for x in (k, v, w)]
        results.append([*evict_keys(*own, tables.to(device), lens, 16, budget, **more), *own])
    for x, y in zip(*results):
        assert torch.equal(x, y)
    with pytest.raises(ValueError, match="budget"):
        evict_keys(*own, tables.to(device), lens, 16, 3)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_weighing_in_wide_tables(device, dtype):
    """Tables padded to far more columns than the requests fill: keys behind a request's end
    get nothing, and the columns' ids are not looked at."""
    lens = [1, 256, 257, 40, 1000]
    k, v, tables = so.pool(lens, 16, 2, 64, dtype, 5, width=2048)
    tables[:, 100:] = 1 << 40
    q = torch.randn(5, 14, 64, generator=torch.Generator().manual_seed(1)).to(dtype)
    weights = torch.zeros(k.shape[0], 2, 16, device=device)
    got = paged_attention_decode_weighted(q.to(device), k.to(device), v.to(device), weights,
                                          tables.to(device), torch.tensor(lens).to(device), 16)
    want = torch.zeros(weights.shape, dtype=torch.float64)
    size = torch.zeros_like(want)
    for i, n in enumerate(lens):
        slot = so.slots(tables[i], n, 16)
        out, bound, p, pb = so.attend(q[i:i + 1], k.view(-1, 2, 64)[slot],
                                      v.view(-1, 2, 64)[slot],
                                      torch.ones(1, n, dtype=torch.bool), 0.125, 0.0, dtype)
        so.assert_within(got[i:i + 1], out, bound, f"request {i}")
        add = p[0].view(2, 7, n).sum(1).T
        want[slot // 16, :, slot % 16] = add
        size[slot // 16, :, slot % 16] = pb[0].view(2, 7, n).sum(1).T + 8 * 2.0 ** -24 * add
    so.assert_within(weights, want, size, "weights")
