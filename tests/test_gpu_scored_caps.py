"""Scored paged attention over the whole range of caps, from one far above the
scores (where the cap changes nothing) to one far below (where all keys weigh
alike), on both kernels.

The bound is scored_oracle.py's, except for the cap: the capped score itself is
off by at most 2^-19 of its own size, however large the cap. (The cap is an odd
polynomial of relative error 5.1e-7 for |x / cap| <= 1/2; above, it is cap (1 - 2 /
(e^(2 y) + 1)), whose error of at most 3.5 2^-23 of the cap is 9e-7 of the score.
2^-19 is 1.9e-6.)
"""

from __future__ import annotations

import pytest
import torch

from mini_llm_runtime_amd.kernels.scored_attention import (
    paged_attention_decode_scored, paged_attention_decode_shared_prefix,
    paged_attention_prefill_scored)
from scored_oracle import assert_within, gather
from test_gpu_scored_attention import padded, pool, queries

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
CAPS = [1e-30, 1e-20, 1e-12, 1e-8, 1e-4, 1e3, 1e5, 1e6, 1e8, 1e12, 1e20, 1e30]


def attend(q, k, v, limit, scale, cap, dtype):
    """q [n, Hq, D] over k, v [N, Hkv, D], the keys below limit [n]: (out, bound) in
    64 bits."""
    group = q.shape[1] // k.shape[1]
    q = q.double().transpose(0, 1)
    k = k.double().transpose(0, 1).repeat_interleave(group, 0)
    v = v.double().transpose(0, 1).repeat_interleave(group, 0)
    seen = torch.arange(k.shape[1])[None] < limit[:, None]
    x = q @ k.mT * scale
    err = (q.shape[-1] + 2) * 2.0 ** -24 * scale * (q.abs() @ k.abs().mT)
    x = cap * torch.tanh(x / cap)
    err = torch.minimum(err, 2 * x.abs().clamp(min=cap)) + 2.0 ** -19 * x.abs()
    p = x.masked_fill(~seen, -torch.inf).softmax(-1)
    worst = err.masked_fill(~seen, 0.0).amax(-1, keepdim=True)
    half = torch.finfo(dtype).eps / 2
    rel = 2 * worst + 2.0 ** -18 + (half if dtype != torch.float32 else 0.0)
    out = p @ v
    bound = half * out.abs().clamp(min=torch.finfo(dtype).tiny) + rel * (p @ v.abs())
    if dtype == torch.float16:  # operands below 2^-14: at most 2^-25 off, of a sum of 1 or more
        bound = bound + 2.0 ** -25 * (seen.double() @ v.abs())
    return out.transpose(0, 1), bound.transpose(0, 1)


@pytest.mark.parametrize("size", [0.0, 1.0, 3.0])
@pytest.mark.parametrize("cap", CAPS)
@pytest.mark.parametrize("hq,hkv,d,bs", [(14, 2, 64, 16), (8, 2, 128, 16), (6, 2, 64, 24)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_caps(device, dtype, hq, hkv, d, bs, cap, size):
    """Single tokens, a chunk of many rows and one of few, and a shared prefix; in
    block sizes of 24 all on the kernel of few rows."""
    n, m = 200, 9
    k, v, (table,) = pool([n], hkv, d, bs, dtype, 71)
    q = queries(n, hq, d, dtype, 72, size)
    kk, vv = gather(k, table, n, bs), gather(v, table, n, bs)
    limit = torch.arange(1, n + 1)
    want, bound = attend(q, kk, vv, limit, d ** -0.5, cap, dtype)
    qd, kd, vd, bt = q.to(device), k.to(device), v.to(device), padded([table]).to(device)
    lens = torch.tensor([n], device=device)

    got = paged_attention_decode_scored(qd[n - 1:], kd, vd, bt, lens, bs, softcap=cap)
    assert_within(got, want[n - 1:], bound[n - 1:], "one token")
    got = paged_attention_prefill_scored(qd, kd, vd, bt, torch.tensor([0, n], device=device), lens,
                                         bs, softcap=cap)
    assert_within(got, want, bound, "a long chunk")
    got = paged_attention_prefill_scored(qd[n - m:], kd, vd, bt,
                                         torch.tensor([0, m], device=device), lens, bs, softcap=cap)
    assert_within(got, want[n - m:], bound[n - m:], "a short chunk")
    # All tokens as requests of one prefix: their own keys are those past it.
    prefix = 150
    rows = torch.arange(prefix - 1, n)
    got = paged_attention_decode_shared_prefix(
        qd[rows.to(device)], kd, vd, bt[0], prefix, bt.expand(len(rows), -1),
        (rows + 1).to(device), bs, softcap=cap)
    assert_within(got, want[rows], bound[rows], "a shared prefix")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scale", [1e12, -1e12, 1e-12])
@pytest.mark.parametrize("d", [64, 128])
def test_zero_scores_at_the_ends_of_cap_and_scale(device, dtype, scale, d):
    """Queries of zero: every visible key weighs the same, on the kernel of many rows."""
    n, bs = 200, 16
    k, v, (table,) = pool([n], 2, d, bs, dtype, 73)
    q = torch.zeros(n, 6, d, dtype=dtype)
    for cap in (1e-30, 1e30):
        want, bound = attend(q, gather(k, table, n, bs), gather(v, table, n, bs),
                             torch.arange(1, n + 1), abs(scale), cap, dtype)
        got = paged_attention_prefill_scored(
            q.to(device), k.to(device), v.to(device), padded([table]).to(device),
            torch.tensor([0, n], device=device), torch.tensor([n], device=device), bs, softcap=cap,
            scale=scale)
        assert_within(got, want, bound, f"cap {cap}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (8, 2, 128)])
def test_one_score_near_a_large_cap(device, dtype, hq, hkv, d):
    """A key whose score with one query is most of the cap, among ordinary ones: the
    other queries keep the accuracy of theirs."""
    n, bs, cap = 200, 16, 1e6
    k, v, (table,) = pool([n], hkv, d, bs, dtype, 74)
    q = queries(n, hq, d, dtype, 75, 2.0)
    q[:, :, 0] = 0.0
    q[90, :, 0] = 400.0
    k[table[20 // bs], 20 % bs, :, 0] = 7e5 * d ** 0.5 / 400.0
    want, bound = attend(q, gather(k, table, n, bs), gather(v, table, n, bs),
                         torch.arange(1, n + 1), d ** -0.5, cap, dtype)
    qd, kd, vd, bt = q.to(device), k.to(device), v.to(device), padded([table]).to(device)
    for first in (0, 88):  # a chunk of many rows, and its last rows
        rows = slice(first, min(n, first + (5 if first else n)))
        ctx = rows.stop
        got = paged_attention_prefill_scored(
            qd[rows], kd, vd, bt, torch.tensor([0, ctx - first], device=device),
            torch.tensor([ctx], device=device), bs, softcap=cap)
        assert_within(got, want[rows], bound[rows], f"rows from {first}")
