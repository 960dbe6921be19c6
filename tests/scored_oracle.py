"""Scored paged attention in 64 bits on the CPU, with a bound on what FP32
arithmetic and 16-bit operands may change of each output element.

For weights p_j = exp(x_j - m) / l and u = eps / 2 of the type:
- the score x_j: a dot product of D terms in FP32 is off by at most
  (D + 2) 2^-24 scale sum |q k|; scaling, the cap (2^-21 of it), the bias and
  the exponent's argument add 2^-21 (|x| + |bias|);
- a weight changes by twice the largest such error (itself and the sum l), and
  by one rounding u as a 16-bit operand; fp16 operands below 2^-14 are off by
  2^-25 instead;
- the sums of P V and l, in FP32 over up to N keys, by N 2^-24 at most, and far
  less in blocks: 2^-18 covers the N of these tests;
- the result is rounded once: u of its value (of the smallest normal number).
"""

from __future__ import annotations

import torch


def attend(q, k, v, pos, limit, scale, cap=0.0, slopes=None, dtype=torch.float32):
    """q [n, Hq, D] at positions pos [n] over keys [N, Hkv, D], those below
    limit [n]: (out, bound), both [n, Hq, D] in 64 bits."""
    n, hq, d = q.shape
    hkv = k.shape[1]
    group = hq // hkv
    q, k, v = q.double(), k.double(), v.double()
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    key = torch.arange(k.shape[0])
    seen = key[None] < limit[:, None]
    if k.shape[0] == 0:
        return out, bound
    half = torch.finfo(dtype).eps / 2
    for h in range(hq):
        kh, vh = k[:, h // group], v[:, h // group]
        # What is hidden may hold anything: it takes no part, not even times 0.
        used = seen.any(0)
        kh = torch.where(used[:, None], kh, 0.0)
        vh = torch.where(used[:, None], vh, 0.0)
        x = q[:, h] @ kh.T * scale
        err = (d + 2) * 2.0 ** -24 * abs(scale) * (q[:, h].abs() @ kh.abs().T)
        if cap:
            x = cap * torch.tanh(x / cap)
            err = err + 2.0 ** -21 * cap
        bias = 0.0
        if slopes is not None:
            bias = float(slopes[h]) * (pos[:, None] - key[None]).abs().double()
            x = x - bias
        err = err + 2.0 ** -21 * (x.abs() + bias)
        x = x.masked_fill(~seen, -torch.inf)
        m = x.amax(-1, keepdim=True)
        w = torch.where(seen, (x - m).exp(), 0.0)
        l = w.sum(-1, keepdim=True)
        worst = err.masked_fill(~seen, 0.0).amax(-1, keepdim=True)
        p = w / l
        rel = 2 * worst + 2.0 ** -18 + (half if dtype != torch.float32 else 0.0)
        clean = torch.where(vh.isfinite(), vh, 0.0)
        o = p @ clean
        size = p @ clean.abs()
        extra = 0.0
        if dtype == torch.float16:
            extra = 2.0 ** -25 * (seen.double() @ clean.abs()) / l
        empty = ~seen.any(-1)
        # Rows that see a V that is not finite: NaN or infinite there.
        for j in (~vh.isfinite()).any(-1).nonzero().flatten().tolist():
            rows = seen[:, j].nonzero().flatten()
            o[rows] = o[rows] + p[rows, j, None] * torch.where(vh[j].isfinite(), 0.0, vh[j])
        o[empty] = 0.0
        out[:, h] = o
        tiny = torch.finfo(dtype).tiny
        bound[:, h] = torch.where(empty[:, None], 0.0,
                                  half * o.abs().clamp(min=tiny) + rel * size + extra)
    return out, bound


def gather(cache, table, count, block_size):
    """Rows [0, count) of one sequence: [count, Hkv, D]."""
    at = torch.arange(count)
    block = torch.as_tensor(table)[at // block_size] if count else at
    return cache[block, at % block_size]


def assert_within(got, want, bound, what=""):
    got = got.double().cpu()
    same = (got == want) | (got.isnan() & want.isnan())
    err = (got - want).abs() - bound
    bad = ~same & ~(err <= 0)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} past the bound, first at "
                           f"{bad.nonzero()[0].tolist()}: {got[bad][0]} for {want[bad][0]}, "
                           f"bound {bound[bad][0]}")
