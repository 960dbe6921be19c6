"""paged_attention_decode_scored, paged_attention_prefill_scored and
paged_attention_decode_shared_prefix against the definition in 64 bits
(scored_oracle.py, which derives the bound of each element)."""

from __future__ import annotations

import math

import pytest
import torch

from mini_llm_runtime_amd.kernels.scored_attention import (
    paged_attention_decode_scored, paged_attention_decode_shared_prefix,
    paged_attention_prefill_scored)
from scored_oracle import assert_within, attend, gather

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def pool(lens, hkv, d, bs, dtype, seed, stale=math.nan):
    """(k, v, tables): rows of no sequence, in used blocks too, hold `stale`."""
    gen = torch.Generator().manual_seed(seed)
    need = [-(-n // bs) for n in lens]
    blocks = sum(need) + 3
    perm = torch.randperm(blocks, generator=gen).tolist()
    k = torch.full((blocks, bs, hkv, d), stale, dtype=dtype)
    v = k.clone()
    tables, at = [], 0
    for n, c in zip(lens, need):
        table = perm[at:at + c]
        at += c
        for i, b in enumerate(table):
            rows = min(bs, n - i * bs)
            k[b, :rows] = torch.randn(rows, hkv, d, generator=gen).to(dtype)
            v[b, :rows] = torch.randn(rows, hkv, d, generator=gen).to(dtype)
        tables.append(table)
    return k, v, tables


def padded(tables, extra=0):
    width = max((len(t) for t in tables), default=0) + extra
    return torch.tensor([t + [-1] * (width - len(t)) for t in tables], dtype=torch.long).view(
        len(tables), width)


def slopes_of(hq):
    return 2.0 ** (-8.0 * torch.arange(1, hq + 1) / hq)


def queries(n, hq, d, dtype, seed, size=1.0):
    gen = torch.Generator().manual_seed(seed)
    return (size * torch.randn(n, hq, d, generator=gen)).to(dtype)


SCORES = [dict(), dict(cap=20.0), dict(alibi=True), dict(cap=5.0, alibi=True, scale=0.3)]


def kwargs_of(score, hq, d, device=None):
    """(arguments of the call, of the oracle)."""
    slopes = slopes_of(hq) if score.get("alibi") else None
    scale = score.get("scale", d ** -0.5)
    call = dict(softcap=score.get("cap", 0.0), scale=scale,
                alibi_slopes=None if slopes is None else slopes.to(device))
    return call, dict(scale=scale, cap=score.get("cap", 0.0), slopes=slopes)


def decode_case(device, lens, hq, hkv, d, bs, dtype, score, seed=0, size=1.0, extra=0, **more):
    k, v, tables = pool(lens, hkv, d, bs, dtype, seed)
    q = queries(len(lens), hq, d, dtype, seed + 1, size)
    call, ref = kwargs_of(score, hq, d, device)
    got = paged_attention_decode_scored(
        q.to(device), k.to(device), v.to(device), padded(tables, extra).to(device),
        torch.tensor(lens, device=device), bs, **call, **more)
    for b, n in enumerate(lens):
        want, bound = attend(q[b:b + 1], gather(k, tables[b], n, bs), gather(v, tables[b], n, bs),
                             torch.tensor([n - 1]), torch.tensor([n]), dtype=dtype, **ref)
        assert_within(got[b:b + 1], want, bound, f"request {b} of {n} keys")
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("score", SCORES, ids=str)
@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (28, 4, 128), (4, 2, 16), (8, 2, 96),
                                      (12, 12, 64), (10, 2, 80), (32, 1, 32), (3, 3, 8)])
def test_decode(device, dtype, score, hq, hkv, d):
    decode_case(device, [1, 16, 17, 130, 515, 2049], hq, hkv, d, 16, dtype, score)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bs", [1, 3, 8, 24, 32, 48, 256])
def test_decode_block_sizes(device, dtype, bs):
    decode_case(device, [5, 64, 700], 6, 2, 64, bs, dtype, dict(cap=30.0, alibi=True))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lens,extra", [([9000], 0), ([20000, 3], 0), ([40] * 70, 0),
                                        ([33, 700, 5], 3000)])
def test_decode_splits(device, dtype, lens, extra):
    """One long request over many splits; many short; a table far wider than
    its contexts."""
    decode_case(device, lens, 14, 2, 64, 16, dtype, dict(cap=50.0), extra=extra)


@pytest.mark.parametrize("dtype", DTYPES)
def test_decode_large_scores(device, dtype):
    """Scores of several hundred: one key takes nearly all weight, and the cap
    flattens them."""
    decode_case(device, [300, 40], 4, 2, 64, 16, dtype, dict(), size=40.0)
    decode_case(device, [300, 40], 4, 2, 64, 16, dtype, dict(cap=1e4), size=40.0)
    decode_case(device, [300, 40], 4, 2, 64, 16, dtype, dict(cap=0.5), size=40.0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_decode_padded_rows_and_missing_blocks(device, dtype):
    """Rows of length 0 give zeros; keys in blocks out of range are not seen."""
    lens, bs, hq, hkv, d = [40, 0, 300, 0], 16, 6, 2, 64
    k, v, tables = pool([40, 0, 300, 0], hkv, d, bs, dtype, 3)
    q = queries(4, hq, d, dtype, 4)
    bt = padded(tables)
    bt[2, 3], bt[2, 7] = -1, 10 ** 9
    got = paged_attention_decode_scored(q.to(device), k.to(device), v.to(device), bt.to(device),
                                        torch.tensor(lens, device=device), bs, softcap=10.0,
                                        validate=False)
    assert (got[1] == 0).all() and (got[3] == 0).all()
    keep = torch.ones(300, dtype=torch.bool)
    keep[48:64] = keep[112:128] = False
    kk, vv = gather(k, tables[2], 300, bs)[keep], gather(v, tables[2], 300, bs)[keep]
    want, bound = attend(q[2:3], kk, vv, torch.tensor([299]), torch.tensor([300]), d ** -0.5, 10.0,
                         dtype=dtype)
    assert_within(got[2:3], want, bound)


def test_decode_strides_out_and_lists(device):
    lens, bs = [70, 200], 16
    k, v, tables = pool(lens, 2, 64, bs, torch.bfloat16, 5)
    q = queries(2, 6, 64, torch.bfloat16, 6).to(device)
    k, v = k.to(device), v.to(device)
    bt, sl = padded(tables).to(device), torch.tensor(lens, device=device)
    want = paged_attention_decode_scored(q, k, v, bt, sl, bs, softcap=9.0)
    wide = torch.zeros(2, 6, 100, dtype=q.dtype, device=device)
    wide[:, :, 1:65] = q  # rows at odd addresses
    turned = q.transpose(0, 1).contiguous().transpose(0, 1)
    big = torch.full((2, 8, 80), 5.0, dtype=q.dtype, device=device)
    wider = torch.full((2, 2 * bt.shape[1]), -1, device=device)
    wider[:, ::2] = bt
    for got in (paged_attention_decode_scored(wide[:, :, 1:65], k, v, bt, sl, bs, softcap=9.0),
                paged_attention_decode_scored(turned, k, v, bt, sl.int(), bs, softcap=9.0),
                paged_attention_decode_scored(q, k, v, bt.int(), lens, bs, softcap=9.0),
                paged_attention_decode_scored(q, k, v, wider[:, ::2], sl, bs, softcap=9.0),
                paged_attention_decode_scored(q, k, v, bt, sl, bs, softcap=9.0,
                                              out=big[:, 1:7, 3:67])):
        assert torch.equal(got, want)
    assert (big[:, 0] == 5).all() and (big[:, 7] == 5).all()
    assert (big[:, :, :3] == 5).all() and (big[:, :, 67:] == 5).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_visible_values_that_are_not_finite_stay_in_their_request(device, dtype):
    lens, bs, hq, hkv, d = [90, 200, 30], 16, 4, 2, 64
    k, v, tables = pool(lens, hkv, d, bs, dtype, 7)
    v[tables[1][2], 5, 1] = math.nan
    q = queries(3, hq, d, dtype, 8)
    got = paged_attention_decode_scored(q.to(device), k.to(device), v.to(device),
                                        padded(tables).to(device),
                                        torch.tensor(lens, device=device), bs)
    nan = got.isnan()
    assert nan[1, 2:].all() and not nan[1, :2].any() and not nan[0].any() and not nan[2].any()


# ---------------------------------------------------------------------------
# Prefill
# ---------------------------------------------------------------------------
def prefill_case(device, chunks, hq, hkv, d, bs, dtype, score, ahead=None, seed=0, **more):
    """chunks: [(past, queries)]."""
    lens = [p + n for p, n in chunks]
    k, v, tables = pool(lens, hkv, d, bs, dtype, seed)
    total = sum(n for _, n in chunks)
    q = queries(total, hq, d, dtype, seed + 1)
    qsl = torch.tensor([0] + [n for _, n in chunks]).cumsum(0)
    call, ref = kwargs_of(score, hq, d, device)
    got = paged_attention_prefill_scored(
        q.to(device), k.to(device), v.to(device), padded(tables).to(device), qsl.to(device),
        torch.tensor(lens, device=device), bs, **call,
        prefix_lens=None if ahead is None else torch.tensor(ahead, device=device), **more)
    for s, (past, n) in enumerate(chunks):
        pos = past + torch.arange(n)
        limit = pos + 1
        if ahead is not None:
            limit = limit.clamp(min=ahead[s])
        rows = slice(int(qsl[s]), int(qsl[s + 1]))
        want, bound = attend(q[rows], gather(k, tables[s], past + n, bs),
                             gather(v, tables[s], past + n, bs), pos, limit, dtype=dtype, **ref)
        assert_within(got[rows], want, bound, f"sequence {s}: {past} past, {n} queries")
    return got


CHUNKS = [(0, 1), (0, 70), (129, 33), (400, 1), (7, 300), (0, 0), (50, 200)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("score", SCORES, ids=str)
@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (4, 1, 128), (4, 2, 16), (8, 2, 96),
                                      (3, 3, 64), (10, 2, 80)])
def test_prefill(device, dtype, score, hq, hkv, d):
    prefill_case(device, CHUNKS, hq, hkv, d, 16, dtype, score)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (8, 2, 128), (6, 2, 48)])
def test_prefill_prefix_seen_whole(device, dtype, hq, hkv, d):
    ahead = [1, 40, 162, 0, 306, 0, 100]
    prefill_case(device, CHUNKS, hq, hkv, d, 16, dtype, dict(alibi=True), ahead=ahead)
    prefill_case(device, CHUNKS, hq, hkv, d, 16, dtype, dict(cap=15.0), ahead=ahead,
                 max_query_len=1000)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bs", [1, 8, 24, 32, 64])
def test_prefill_block_sizes(device, dtype, bs):
    prefill_case(device, [(30, 90), (0, 129)], 6, 2, 64, bs, dtype, dict(cap=30.0, alibi=True),
                 ahead=[60, 100])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_prefill_few_queries_after_many_keys(device, dtype, d):
    prefill_case(device, [(6000, 20)], 4, 2, d, 16, dtype, dict(cap=50.0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_prefill_values_that_are_not_finite(device, dtype, d, value):
    """A V that is not finite reaches the queries that see its key, no others."""
    lens, bs, hq, hkv = [150, 80], 16, 4, 2
    k, v, tables = pool(lens, hkv, d, bs, dtype, 11)
    v[tables[0][100 // bs], 100 % bs, 0, 5] = value
    v[tables[0][149 // bs], 149 % bs, 1] = value
    q = queries(230, hq, d, dtype, 12)
    got = paged_attention_prefill_scored(
        q.to(device), k.to(device), v.to(device), padded(tables).to(device),
        torch.tensor([0, 150, 230], device=device), torch.tensor(lens, device=device), bs,
        softcap=8.0)
    bad = ~torch.isfinite(got.cpu())
    want = torch.zeros_like(bad)
    want[100:150, :2, 5] = True
    want[149, 2:] = True
    assert torch.equal(bad, want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_prefill_leaves_other_rows(device, dtype):
    lens, bs = [20, 35], 16
    k, v, tables = pool(lens, 2, 64, bs, dtype, 13)
    q = queries(70, 4, 64, dtype, 14).to(device)
    out = torch.full((70, 4, 64), 3.0, dtype=dtype, device=device)
    paged_attention_prefill_scored(q, k.to(device), v.to(device), padded(tables).to(device),
                                   torch.tensor([5, 25, 60], device=device),
                                   torch.tensor(lens, device=device), bs, validate=False,
                                   max_query_len=35, out=out)
    assert (out[:5] == 3).all() and (out[60:] == 3).all() and (out[5:60] != 3).any(-1).all()


def test_prefill_equals_decode_on_single_tokens(device):
    """One token a sequence through either call: the same definition."""
    lens = [1, 40, 333]
    k, v, tables = pool(lens, 2, 64, 16, torch.float32, 15)
    q = queries(3, 6, 64, torch.float32, 16).to(device)
    k, v, bt = k.to(device), v.to(device), padded(tables).to(device)
    sl = torch.tensor(lens, device=device)
    a = paged_attention_prefill_scored(q, k, v, bt, torch.arange(4, device=device), sl, 16,
                                       softcap=20.0)
    b = paged_attention_decode_scored(q, k, v, bt, sl, 16, softcap=20.0)
    assert (a - b).abs().max() <= 2.0 ** -17 * b.abs().max()


# ---------------------------------------------------------------------------
# Shared prefix
# ---------------------------------------------------------------------------
def shared_case(device, prefix, owns, hq, hkv, d, bs, dtype, score, seed=0, repeat=False):
    whole = prefix // bs
    lens = [prefix + n for n in owns]
    k, v, tables = pool([prefix] + [n - whole * bs for n in lens], hkv, d, bs, dtype, seed)
    ptable, own = tables[0], tables[1:]
    # Rows of a request's first block that lie before the prefix's end are
    # nobody's: the prefix has them.
    for t in own:
        if t:
            k[t[0], :prefix - whole * bs] = math.nan
            v[t[0], :prefix - whole * bs] = math.nan
    q = queries(len(owns), hq, d, dtype, seed + 1)
    call, ref = kwargs_of(score, hq, d, device)
    head = ptable[:whole] if repeat else [-7] * whole
    bt = padded([head + t for t in own])
    got = paged_attention_decode_shared_prefix(
        q.to(device), k.to(device), v.to(device), torch.tensor(ptable, dtype=torch.long,
                                                               device=device), prefix,
        bt.to(device), torch.tensor(lens, device=device), bs, **call)
    for b, n in enumerate(lens):
        kk = gather(k, ptable, prefix, bs)
        vv = gather(v, ptable, prefix, bs)
        table = [0] * whole + own[b]
        kk = torch.cat([kk, gather(k, table, n, bs)[prefix:]])
        vv = torch.cat([vv, gather(v, table, n, bs)[prefix:]])
        want, bound = attend(q[b:b + 1], kk, vv, torch.tensor([n - 1]), torch.tensor([n]),
                             dtype=dtype, **ref)
        assert_within(got[b:b + 1], want, bound, f"request {b}: {prefix} + {owns[b]} keys")
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("score", SCORES, ids=str)
@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (28, 4, 128), (4, 2, 16), (32, 1, 64),
                                      (8, 2, 96), (3, 3, 40)])
def test_shared_prefix(device, dtype, score, hq, hkv, d):
    shared_case(device, 300, [1, 0, 20, 150, 4, 700, 33], hq, hkv, d, 16, dtype, score)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("prefix", [0, 1, 15, 16, 64, 1000, 2048])
def test_shared_prefix_lengths(device, dtype, prefix):
    shared_case(device, prefix, [1, 40, 130] if prefix == 0 else [0, 1, 40, 130], 14, 2, 64, 16,
                dtype, dict(alibi=True), repeat=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bs", [1, 8, 24, 64])
def test_shared_prefix_block_sizes(device, dtype, bs):
    shared_case(device, 333, [5, 40, 1], 6, 2, 64, bs, dtype, dict(cap=10.0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch", [1, 3, 40])
def test_shared_prefix_batches(device, dtype, batch):
    shared_case(device, 5000, [(7 * i) % 90 for i in range(batch)], 14, 2, 64, 16, dtype, dict())


def test_shared_prefix_of_short_and_padded_requests(device):
    """Unchecked: a request inside the prefix sees its own positions, one of
    length 0 nothing."""
    prefix, bs, dtype = 100, 16, torch.float32
    k, v, tables = pool([prefix], 2, 64, bs, dtype, 21)
    q = queries(3, 6, 64, dtype, 22)
    lens = [60, 0, 100]
    for width in (0, 7):
        got = paged_attention_decode_shared_prefix(
            q.to(device), k.to(device), v.to(device), torch.tensor(tables[0], device=device),
            prefix, torch.full((3, width), -1, device=device), torch.tensor(lens, device=device),
            bs, alibi_slopes=slopes_of(6).to(device), validate=False)
        assert (got[1] == 0).all()
        for b in (0, 2):
            n = lens[b]
            want, bound = attend(q[b:b + 1], gather(k, tables[0], n, bs),
                                 gather(v, tables[0], n, bs), torch.tensor([n - 1]),
                                 torch.tensor([n]), 0.125, 0.0, slopes_of(6), dtype=dtype)
            assert_within(got[b:b + 1], want, bound)


# ---------------------------------------------------------------------------
# Streams and graphs
# ---------------------------------------------------------------------------
def three_calls(device, dtype, seed):
    lens, bs = [300, 900, 40], 16
    k, v, tables = pool([200] + lens, 2, 64, bs, dtype, seed, stale=0.0)
    k, v = k.to(device), v.to(device)
    bt = padded(tables[1:]).to(device)
    sl = torch.tensor(lens, device=device)
    ptable = torch.tensor(tables[0], device=device)
    full = torch.cat([ptable[:12].expand(3, -1), bt], 1)
    q = queries(3, 14, 64, dtype, seed + 1).to(device)
    rows = queries(70, 14, 64, dtype, seed + 2).to(device)
    qsl = torch.tensor([0, 30, 65, 70], device=device)

    def run():
        return (paged_attention_decode_scored(q, k, v, bt, sl, bs, softcap=30.0, validate=False),
                paged_attention_prefill_scored(rows, k, v, bt, qsl, sl, bs, max_query_len=35,
                                               softcap=30.0, validate=False),
                paged_attention_decode_shared_prefix(q, k, v, ptable, 200, full, sl + 192, bs,
                                                     validate=False))

    return run, (q, rows, sl)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_captured_graphs_side_by_side(device, dtype):
    """Two graphs of the same calls, replayed in turn with new queries and
    lengths, equal the eager calls every time."""
    runs = [three_calls(device, dtype, 30), three_calls(device, dtype, 40)]
    graphs, outs = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for run, _ in runs:
            run()
    torch.cuda.current_stream().wait_stream(side)
    for run, _ in runs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(run())
    for i in range(3):
        for run, (q, rows, sl) in runs:
            q.mul_(-0.9)
            rows.mul_(1.1)
            sl.sub_(3)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (run, _), out in zip(runs, outs):
            for a, b in zip(out, run()):
                assert torch.equal(a, b)


def test_two_streams_at_once(device):
    run, _ = three_calls(device, torch.bfloat16, 50)
    want = run()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(4):
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(run())
    torch.cuda.synchronize()
    for out in got:
        for a, b in zip(out, want):
            assert torch.equal(a, b)
