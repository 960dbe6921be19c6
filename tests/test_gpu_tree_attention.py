"""Drafted trees against 64 bits: tree_ancestors and paged_attention_tree."""

from __future__ import annotations

import random

import pytest
import torch

from mini_llm_runtime_amd.kernels.scored_attention import paged_attention_prefill_scored
from mini_llm_runtime_amd.kernels.tree_attention import paged_attention_tree, tree_ancestors

import selection_oracle as so

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def bits_of(sets, words):
    rows = []
    for s in sets:
        value = sum(1 << j for j in s)
        row = [value >> 64 * w & (1 << 64) - 1 for w in range(words)]
        rows.append([x - (1 << 64) if x >> 63 else x for x in row])
    return torch.tensor(rows, dtype=torch.long)


def packed(trees):
    qsl = [0]
    for t in trees:
        qsl.append(qsl[-1] + len(t))
    return torch.tensor(qsl)


def run_case(device, dtype, heads, past, counts, block_size=16, cap=0.0, sets=None, seed=0,
             words=None, change=None, scale=None):
    hq, hkv, d = heads
    rng = random.Random(seed)
    if sets is None:
        sets = [so.paths(so.random_parents(n, rng)) for n in counts]
    lens = [p + n for p, n in zip(past, counts)]
    k, v, tables = so.pool(lens, block_size, hkv, d, dtype, seed + 1)
    total = sum(counts)
    gen = torch.Generator().manual_seed(seed + 2)
    q = torch.randn(total, hq, d, generator=gen).to(dtype)
    if change is not None:
        change(k, v, tables, lens)
    words = words or max(1, -(-max(counts) // 64))
    bits = torch.cat([bits_of(s, words) for s in sets if s] or
                     [torch.zeros(0, words, dtype=torch.long)])
    qsl = packed(sets)
    scale = d ** -0.5 if scale is None else scale
    out = torch.full((total + 2, hq, d), 7.0, dtype=dtype, device=device)
    got = paged_attention_tree(
        q.to(device), k.to(device), v.to(device), tables.to(device), qsl.to(device),
        torch.tensor(lens).to(device), bits.to(device), block_size, softcap=cap, scale=scale,
        out=out[:total])
    torch.cuda.synchronize()
    assert (out[total:] == 7.0).all()
    for i, n in enumerate(lens):
        if counts[i] == 0:
            continue
        slot = so.slots(tables[i], n, block_size)
        seen = torch.zeros(counts[i], n, dtype=torch.bool)
        seen[:, :n - counts[i]] = True
        for r, s in enumerate(sets[i]):
            for j in s:
                if j < counts[i]:
                    seen[r, n - counts[i] + j] = True
        rows = slice(int(qsl[i]), int(qsl[i + 1]))
        want, bound, _, _ = so.attend(q[rows], k.view(-1, hkv, d)[slot], v.view(-1, hkv, d)[slot],
                                      seen, scale, cap, dtype)
        so.assert_within(got[rows], want, bound, f"sequence {i}")
    return got


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("heads", [(14, 2, 64), (8, 2, 128), (4, 4, 96), (6, 2, 40), (16, 1, 16)])
def test_trees(device, dtype, heads):
    run_case(device, dtype, heads, [0, 3, 61, 200], [5, 1, 17, 40])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("count", [1, 2, 15, 16, 31, 63, 64, 65, 100, 130])
def test_tree_sizes_and_edges_of_words(device, dtype, count):
    """Trees that start and end at every place of a word, a tile and a block."""
    run_case(device, dtype, (7, 1, 64), [0, 1, 63, 64, 77], [count] * 5, seed=count)


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("block_size", [1, 3, 8, 32, 64, 24])
def test_block_sizes(device, dtype, block_size):
    run_case(device, dtype, (4, 2, 64), [0, 30, 129], [9, 20, 33], block_size=block_size)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_long_prefix_in_splits(device, dtype):
    run_case(device, dtype, (14, 2, 64), [4000], [12])
    run_case(device, dtype, (8, 2, 128), [2500, 10], [24, 3])


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("cap", [5.0, 50.0])
def test_capped(device, dtype, cap):
    run_case(device, dtype, (14, 2, 64), [100, 7], [33, 6], cap=cap)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_negative_scale(device, dtype):
    run_case(device, dtype, (14, 2, 64), [100, 7], [33, 6], scale=-0.2)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("count", [4, 40])
def test_rows_that_see_nothing(device, dtype, count):
    """Empty rows, with and without keys before the drafted ones: zeros where there are none."""
    sets = [[set() if i % 3 == 0 else {i, 0} for i in range(count)] for _ in range(2)]
    got = run_case(device, dtype, (14, 2, 64), [0, 50], [count] * 2, sets=sets)
    assert (got[0] == 0).all() and (got[3] == 0).all() and (got[count] != 0).any()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_any_set_of_bits(device, dtype):
    """Not a tree's: later tokens seen, own ones not; bits past the tokens count for nothing."""
    rng = random.Random(3)
    sets = [[{j for j in range(n + 20) if rng.random() < 0.4} for _ in range(n)] for n in (37, 70)]
    run_case(device, dtype, (14, 2, 64), [20, 130], [37, 70], sets=sets, words=2)


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("count", [6, 50])
def test_hidden_values_that_are_not_finite(device, dtype, count):
    """Node 1 holds NaN and infinities: only the rows that see it meet them."""
    sets = [so.paths([-1] + [0] * (count // 2) + [1] * (count - count // 2 - 1))]

    def change(k, v, tables, lens):
        at = lens[0] - count + 1
        block = tables[0, at // 16]
        v[block, at % 16, :, ::2] = float("nan")
        v[block, at % 16, :, 1::4] = float("inf")

    run_case(device, dtype, (14, 2, 64), [30], [count], sets=sets, change=change)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("count", [6, 50])
def test_hidden_keys_that_are_not_finite(device, dtype, count):
    """A key that no row sees may hold anything, in K and in V."""
    parents = [-1, -1] + [0] * (count - 2)
    sets = [[s - {1} for s in so.paths(parents)]]

    def change(k, v, tables, lens):
        at = lens[0] - count + 1
        block = tables[0, at // 16]
        k[block, at % 16] = float("nan")
        v[block, at % 16] = float("nan")

    got = run_case(device, dtype, (14, 2, 64), [30], [count], sets=sets, change=change)
    assert got.isfinite().all()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_chain_is_causal(device, dtype):
    """A chain of drafted tokens is a prefill chunk: both are within the bound of the exact
    result, hence within twice that of each other."""
    counts, past = [33, 5], [70, 200]
    lens = [p + n for p, n in zip(past, counts)]
    k, v, tables = so.pool(lens, 16, 2, 64, dtype, 5)
    q = torch.randn(sum(counts), 14, 64, generator=torch.Generator().manual_seed(1)).to(dtype)
    qsl = torch.tensor([0, 33, 38]).to(device)
    parents = torch.tensor([*range(-1, 32), *range(-1, 4)]).to(device)
    args = [x.to(device) for x in (q, k, v, tables)]
    ctx = torch.tensor(lens).to(device)
    got = paged_attention_tree(*args, qsl, ctx, tree_ancestors(parents, qsl, 33), 16)
    want = paged_attention_prefill_scored(*args, qsl, ctx, 16).double().cpu()
    for i, n in enumerate(lens):
        slot = so.slots(tables[i], n, 16)
        rows = slice(sum(counts[:i]), sum(counts[:i + 1]))
        seen = torch.arange(n) <= torch.arange(past[i], n)[:, None]
        _, bound, _, _ = so.attend(q[rows], k.view(-1, 2, 64)[slot], v.view(-1, 2, 64)[slot],
                                   seen, 0.125, 0.0, dtype)
        so.assert_within(got[rows], want[rows], 2 * bound)


def test_strides_and_padding(device):
    """q as a view of packed q, k and v rows, an out with wide rows, an empty sequence, and
    metadata rows that the packed tokens do not reach."""
    counts, past = [4, 0, 20], [10, 30, 100]
    lens = [p + n for p, n in zip(past, counts)]
    k, v, tables = so.pool(lens, 16, 2, 64, BF, 5)
    wide = torch.randn(24, 18 * 64, generator=torch.Generator().manual_seed(1)).to(BF).to(device)
    q = wide[:, :14 * 64].view(24, 14, 64)
    sets = [so.paths(so.random_parents(n, random.Random(n))) for n in counts]
    bits = torch.cat([bits_of(s, 1) for s in sets if s]).to(device)
    args = (k.to(device), v.to(device), tables.to(device), packed(sets).to(device),
            torch.tensor(lens).to(device))
    want = paged_attention_tree(q.contiguous(), *args, bits, 16)
    out = torch.zeros(24, 14, 100, dtype=BF, device=device)
    got = paged_attention_tree(q, *args, bits, 16, out=out[..., :64])
    assert got.data_ptr() == out.data_ptr()
    torch.testing.assert_close(got, want, rtol=0, atol=0)
    assert (out[..., 64:] == 0).all()
    # Words of a wider mask, and int32 metadata.
    bits3 = torch.cat([bits, torch.full((24, 2), -1, device=device)], 1)[:, :3]
    got = paged_attention_tree(q, args[0], args[1], args[2].int(), args[3].int(), args[4].int(),
                               bits3, 16)
    torch.testing.assert_close(got, want, rtol=0, atol=0)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("count", [5, 40])
def test_a_bound_past_the_words(device, dtype, count):
    """max_query_len bounds the sequences from above: one past the bits of the words is taken
    as long as no sequence is so long."""
    lens = [count + 30] * 3
    k, v, tables = so.pool(lens, 16, 2, 64, dtype, 5)
    q = torch.randn(3 * count, 14, 64, generator=torch.Generator().manual_seed(1)).to(dtype)
    sets = [so.paths(so.random_parents(count, random.Random(i))) for i in range(3)]
    bits = torch.cat([bits_of(s, 1) for s in sets]).to(device)
    args = [x.to(device) for x in (q, k, v, tables, packed(sets), torch.tensor(lens))]
    for most in (count, 65, 1 << 40):
        got = paged_attention_tree(*args, bits, 16, max_query_len=most)
        for i, s in enumerate(sets):
            seen = torch.zeros(count, lens[i], dtype=torch.bool)
            seen[:, :30] = True
            for r, path in enumerate(s):
                seen[r, [30 + j for j in path]] = True
            slot, rows = so.slots(tables[i], lens[i], 16), slice(i * count, (i + 1) * count)
            want, bound, _, _ = so.attend(q[rows], k.view(-1, 2, 64)[slot],
                                          v.view(-1, 2, 64)[slot], seen, 0.125, 0.0, dtype)
            so.assert_within(got[rows], want, bound, f"bound {most}, sequence {i}")


@pytest.mark.parametrize("dtype", [BF, F32])
def test_bad_blocks_are_masked(device, dtype):
    """With validate=False a block id out of range hides its keys."""
    k, v, tables = so.pool([100], 16, 2, 64, dtype, 5)
    q = torch.randn(40, 14, 64, generator=torch.Generator().manual_seed(1)).to(dtype)
    sets = so.paths(so.random_parents(40, random.Random(1)))
    bits = bits_of(sets, 1)
    seen = torch.zeros(40, 100, dtype=torch.bool)
    seen[:, :60] = True
    for r, s in enumerate(sets):
        seen[r, [60 + j for j in s]] = True
    slot = so.slots(tables[0], 100, 16)
    for at, bad in ((1, -5), (3, 1 << 40)):
        tables[0, at] = bad
        seen[:, 16 * at:16 * at + 16] = False
    got = paged_attention_tree(q.to(device), k.to(device), v.to(device), tables.to(device),
                               torch.tensor([0, 40]).to(device), torch.tensor([100]).to(device),
                               bits.to(device), 16, validate=False, max_query_len=40)
    want, bound, _, _ = so.attend(q, k.view(-1, 2, 64)[slot], v.view(-1, 2, 64)[slot], seen,
                                  64 ** -0.5, 0.0, dtype)
    so.assert_within(got, want, bound)


@pytest.mark.parametrize("counts", [[1], [5, 0, 64, 1], [65, 130, 300], [4096],
                                    [700, 4000]])
def test_ancestors(device, counts):
    rng = random.Random(sum(counts))
    parents = [so.random_parents(n, rng) for n in counts]
    words = -(-max(counts) // 64)
    got = tree_ancestors(torch.tensor(sum(parents, [])).to(device),
                         packed(parents).to(device), max(counts))
    want = torch.cat([bits_of(so.paths(p), words) for p in parents if p])
    assert torch.equal(got.cpu(), want)


def test_ancestors_of_long_chains(device):
    """Chains and circles of the most tokens that a tree may have, and of more: those past
    it are no nodes and have no row."""
    chain, circle = list(range(-1, 4095)), list(range(1, 4096)) + [0]
    more = list(range(-1, 4999))
    qsl = torch.tensor([0, 4096, 8192, 13192, 13195])
    out = torch.full((13195, 64), 5, device=device)
    got = tree_ancestors(torch.tensor(chain + circle + more + [-1, 0, 0]).to(device),
                         qsl.to(device), 4096, out=out).cpu()
    want = bits_of([range(i + 1) for i in range(4096)], 64)
    assert torch.equal(got[:4096], want) and (got[4096:8192] == -1).all()
    assert torch.equal(got[8192:8192 + 4096], want) and (got[8192 + 4096:13192] == 5).all()
    assert torch.equal(got[13192:], bits_of([[0], [0, 1], [0, 2]], 64))


def test_ancestors_of_odd_parents(device):
    """Children before parents, circles, places out of range, and fewer bits than tokens."""
    parents = [2, 0, 4, 3, -7, 6, 5, 99, 1 << 40]
    got = tree_ancestors(torch.tensor(parents).to(device), torch.tensor([0, 9]).to(device), 9)
    assert torch.equal(got.cpu(), bits_of(so.paths(parents), 1))
    chain = list(range(-1, 99))
    got = tree_ancestors(torch.tensor(chain).to(device), torch.tensor([0, 100]).to(device), 64)
    want = bits_of(so.paths(chain), 2)[:, :1]
    assert torch.equal(got.cpu(), want)
    out = torch.full((12, 1), 5, device=device)
    tree_ancestors(torch.tensor(parents + [0] * 3).to(device), torch.tensor([0, 9]).to(device), 9,
                   out=out)
    assert torch.equal(out[:9].cpu(), bits_of(so.paths(parents), 1)) and (out[9:] == 5).all()
