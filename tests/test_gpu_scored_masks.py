"""Scored paged attention where rows of one unit see different keys: values that
are not finite past a request's length, requests shorter than the shared prefix,
and chunks that their contexts do not cover."""

from __future__ import annotations

import math

import pytest
import torch

from mini_llm_runtime_amd.kernels.scored_attention import (
    paged_attention_decode_shared_prefix, paged_attention_prefill_scored)
from scored_oracle import assert_within, attend, gather
from test_gpu_scored_attention import padded, pool, queries

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("lens", [[100, 0, 170, 199, 200], [64, 0], [0, 0, 300],
                                  [100, 0, 170, 199, 250] * 12], ids=len)
@pytest.mark.parametrize("hq,hkv,d,bs", [(6, 2, 64, 16), (14, 2, 64, 24), (8, 2, 128, 16),
                                         (4, 4, 80, 16), (32, 8, 128, 8)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_shared_prefix_values_that_are_not_finite(device, dtype, hq, hkv, d, bs, lens, value):
    """Unchecked: a request inside the prefix sees its own positions only, one of
    length 0 none. V at position 170 of the prefix is not finite."""
    prefix, at, col = 200, 170, 5
    k, v, tables = pool([prefix] + [max(n - prefix // bs * bs, 0) for n in lens], hkv, d, bs,
                        dtype, 81)
    v[tables[0][at // bs], at % bs, 0, col] = value
    q = queries(len(lens), hq, d, dtype, 82)
    bt = padded([[-1] * (prefix // bs) + t for t in tables[1:]], 1)
    got = paged_attention_decode_shared_prefix(
        q.to(device), k.to(device), v.to(device), torch.tensor(tables[0], device=device), prefix,
        bt.to(device), torch.tensor(lens, device=device), bs, softcap=20.0, validate=False).cpu()
    bad = torch.zeros(got.shape, dtype=torch.bool)
    for b, n in enumerate(lens):
        if n == 0:
            assert (got[b] == 0).all()
            continue
        table = tables[0][:prefix // bs] + tables[1 + b]
        kk, vv = gather(k, tables[0], min(n, prefix), bs), gather(v, tables[0], min(n, prefix), bs)
        if n > prefix:
            kk = torch.cat([kk, gather(k, table, n, bs)[prefix:]])
            vv = torch.cat([vv, gather(v, table, n, bs)[prefix:]])
        if n > at:
            bad[b, :hq // hkv, col] = True
            assert torch.isfinite(vv[at, 1:]).all() and not torch.isfinite(vv[at, 0, col])
            vv[at, 0, col] = 0.0
        want, bound = attend(q[b:b + 1], kk, vv, torch.tensor([n - 1]), torch.tensor([n]),
                             d ** -0.5, 20.0, dtype=dtype)
        row = torch.where(bad[b:b + 1], want, got[b:b + 1].double())
        assert_within(row, want, bound, f"request {b} of {n} keys")
    assert torch.equal(~torch.isfinite(got), bad)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (8, 2, 128)])
@pytest.mark.parametrize("seqs", [[(300, 0), (300, 0)], [(300, 40), (70, 70), (300, 0), (200, 3)],
                                  [(150, 0)]], ids=str)
def test_chunks_longer_than_their_context(device, dtype, hq, hkv, d, seqs):
    """Unchecked: rows before position 0 (a chunk of n queries whose context is
    shorter, or a padded one of context 0) see no key and get zeros; the others
    their own keys."""
    bs = 16
    k, v, tables = pool([c for _, c in seqs], hkv, d, bs, dtype, 83)
    total = sum(n for n, _ in seqs)
    q = queries(total, hq, d, dtype, 84)
    qsl = torch.tensor([0] + [n for n, _ in seqs]).cumsum(0)
    out = torch.full(q.shape, 7.0, dtype=dtype, device=device)
    got = paged_attention_prefill_scored(
        q.to(device), k.to(device), v.to(device), padded(tables, 1).to(device), qsl.to(device),
        torch.tensor([c for _, c in seqs], device=device), bs, softcap=20.0, validate=False,
        max_query_len=max(n for n, _ in seqs), out=out)
    for s, (n, c) in enumerate(seqs):
        rows = slice(int(qsl[s]), int(qsl[s + 1]))
        pos = c - n + torch.arange(n)
        want, bound = attend(q[rows], gather(k, tables[s], c, bs), gather(v, tables[s], c, bs),
                             pos, (pos + 1).clamp(min=0), d ** -0.5, 20.0, dtype=dtype)
        assert_within(got[rows], want, bound, f"sequence {s}: {n} queries, context {c}")
