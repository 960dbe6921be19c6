"""Scored paged attention where its kernels change their way: whole units and
splits, many and few units, one round of items and several."""

from __future__ import annotations

import pytest
import torch

from mini_llm_runtime_amd.kernels.scored_attention import (
    paged_attention_decode_scored, paged_attention_prefill_scored)
from scored_oracle import assert_within, attend, gather
from test_gpu_scored_attention import (decode_case, kwargs_of, padded, pool, prefill_case,
                                       queries, shared_case)

pytestmark = pytest.mark.gpu

HALF = [torch.bfloat16, torch.float16]
SCORE = dict(cap=20.0, alibi=True)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (8, 2, 128)])
@pytest.mark.parametrize("columns", [1, 100, 700])
def test_short_contexts_in_wide_tables(device, dtype, hq, hkv, d, columns):
    """What the table could hold asks for splits, what it holds may not."""
    chunks = [(0, 40), (300, 9), (33, 60)]
    lens = [p + n for p, n in chunks]
    k, v, tables = pool(lens, hkv, d, 16, dtype, 61)
    q = queries(109, hq, d, dtype, 62)
    qsl = torch.tensor([0, 40, 49, 109])
    call, ref = kwargs_of(SCORE, hq, d, device)
    got = paged_attention_prefill_scored(
        q.to(device), k.to(device), v.to(device), padded(tables, columns).to(device),
        qsl.to(device), torch.tensor(lens, device=device), 16, **call)
    for s, (past, n) in enumerate(chunks):
        pos = past + torch.arange(n)
        rows = slice(int(qsl[s]), int(qsl[s + 1]))
        want, bound = attend(q[rows], gather(k, tables[s], lens[s], 16),
                             gather(v, tables[s], lens[s], 16), pos, pos + 1, dtype=dtype, **ref)
        assert_within(got[rows], want, bound, f"sequence {s}")


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("chunks", [[(2500, 50), (10, 3), (0, 33), (700, 64)],
                                    [(3000, 150)], [(0, 0), (1999, 33)]], ids=str)
def test_units_of_unlike_length_split(device, dtype, chunks):
    prefill_case(device, chunks, 8, 2, 64, 16, dtype, SCORE)
    prefill_case(device, chunks, 4, 1, 128, 32, dtype, dict(cap=20.0),
                 ahead=[p // 2 for p, _ in chunks])


@pytest.mark.parametrize("dtype", HALF)
def test_more_sequences_than_are_ranked(device, dtype):
    chunks = [(i % 7, 1 + (5 * i) % 12) for i in range(530)]
    prefill_case(device, chunks, 7, 1, 64, 16, dtype, SCORE)


@pytest.mark.parametrize("dtype", HALF)
def test_more_units_than_are_ranked(device, dtype):
    prefill_case(device, [(3, 40), (0, 90), (20, 1)], 7, 1, 64, 16, dtype, SCORE)
    # The same sequences among many that are empty, with room for long ones.
    chunks = [(0, 0)] * 150 + [(3, 40), (0, 90), (20, 1)] + [(0, 0)] * 150
    prefill_case(device, chunks, 7, 1, 64, 16, dtype, SCORE, max_query_len=2000)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hq,hkv,d", [(8, 4, 64), (8, 8, 128)])
def test_decode_of_more_units_than_a_round(device, dtype, hq, hkv, d):
    lens = [1 + (37 * i) % 300 for i in range(150)] + [1500, 2]
    decode_case(device, lens, hq, hkv, d, 16, dtype, SCORE)


@pytest.mark.parametrize("group", [1, 20, 130])
def test_shared_prefix_of_few_rows(device, group):
    """One and two requests: fewer rows than a unit, and a group larger than one."""
    for owns in ([5], [1, 140]):
        shared_case(device, 700, owns, group, 1, 64, 16, torch.bfloat16, SCORE)


@pytest.mark.parametrize("group", [20, 130])
def test_decode_of_large_groups(device, group):
    decode_case(device, [1, 700, 33], 2 * group, 2, 64, 16, torch.float16, SCORE)


def test_longest_chunk_must_be_declared(device):
    k, v, tables = pool([40], 2, 64, 16, torch.bfloat16, 63)
    q = queries(40, 4, 64, torch.bfloat16, 64).to(device)
    args = (q, k.to(device), v.to(device), padded(tables).to(device),
            torch.tensor([0, 40], device=device), torch.tensor([40], device=device), 16)
    with pytest.raises(ValueError, match="longest chunk"):
        paged_attention_prefill_scored(*args, max_query_len=39)
    with pytest.raises(ValueError, match="longest chunk"):
        paged_attention_prefill_scored(*args, max_query_len=0)
    paged_attention_prefill_scored(*args, max_query_len=40)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_empty_table(device, dtype):
    """No block at all: a padded batch whose every row is empty."""
    k, v, _ = pool([16], 2, 64, 16, dtype, 65)
    q = queries(3, 4, 64, dtype, 66).to(device)
    got = paged_attention_decode_scored(
        q, k.to(device), v.to(device), torch.empty(3, 0, dtype=torch.long, device=device),
        torch.zeros(3, dtype=torch.long, device=device), 16, validate=False)
    assert torch.equal(got, torch.zeros_like(got))
