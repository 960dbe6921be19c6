"""qk_norm_rope_write (mlr_qk_norm_rope_write) against its formulas in 64 bits.

Tolerance per element: the one rounding of the result, eps / 2 of its value
(of the smallest normal number where the value is below it: subnormal numbers
are eps * tiny apart, 2^-24 in fp16, so their rounding is off by half of that),
plus the FP32 arithmetic before it. The norm's sum of D <= 256 products, its
root and three products are off by less than 2^-20 of the value, and the angle
by 2^-25 turns and one rounding of sine and cosine (together under 2^-21), so
2^-19 (|lo| + |hi|) of the rotated pair covers both.
"""

from __future__ import annotations

import math

import pytest
import torch

from mini_llm_runtime_amd.kernels.pre_attention import qk_norm_rope_write, rotary_frequencies

pytestmark = pytest.mark.gpu

BS = 16


def reference(qkv, positions, inv_freq, hq, hkv, d, qw, kw, eps, inter, factor):
    """(q, k, v) in 64 bits with the pair magnitudes |lo| + |hi| of q and k."""
    x = qkv.double().view(-1, hq + 2 * hkv, d)
    rot = 2 * inv_freq.numel()
    angle = positions.double()[:, None] * inv_freq.float().double()[None]
    cos, sin = (factor * angle.cos())[:, None], (factor * angle.sin())[:, None]
    out = []
    for part, w in ((x[:, :hq], qw), (x[:, hq:hq + hkv], kw)):
        n = part
        if w is not None:
            n = part * w.double() / torch.sqrt((part * part).mean(-1, keepdim=True) + eps)
        res, mag = n.clone(), n.abs()
        a, b = ((slice(0, rot, 2), slice(1, rot, 2)) if inter
                else (slice(0, rot // 2), slice(rot // 2, rot)))
        lo, hi = n[..., a], n[..., b]
        res[..., a], res[..., b] = lo * cos - hi * sin, hi * cos + lo * sin
        mag[..., a] = mag[..., b] = (lo.abs() + hi.abs()) * factor
        out.append((res, mag))
    return out[0], out[1], x[:, hq + hkv:]


def make(device, tokens, hq, hkv, d, rot, dtype, seed, far=40000, norm=True, i32=False):
    gen = torch.Generator().manual_seed(seed)
    blocks = tokens // BS + 3
    t = dict(
        qkv=torch.randn(tokens, (hq + 2 * hkv) * d, generator=gen).to(dtype),
        positions=torch.randint(0, far, (tokens,), generator=gen),
        inv_freq=rotary_frequencies(rot, 1e6)[0],
        k=torch.randn(blocks, BS, hkv, d, generator=gen).to(dtype),
        v=torch.randn(blocks, BS, hkv, d, generator=gen).to(dtype),
        slots=torch.randperm(blocks * BS, generator=gen)[:tokens],
        qw=(1 + 0.2 * torch.randn(d, generator=gen)).to(dtype) if norm else None,
        kw=(1 + 0.2 * torch.randn(d, generator=gen)).to(dtype) if norm else None)
    if i32:
        t["slots"] = t["slots"].int()
    return {n: None if x is None else x.to(device) for n, x in t.items()}


def check(t, hq, hkv, d, inter=False, factor=1.0, eps=1e-6, qkv=None, out=None, skipped=()):
    """Runs the call and compares q and the whole caches."""
    dtype = t["qkv"].dtype
    (q, qm), (k, km), v = reference(t["qkv"].cpu(), t["positions"].cpu(), t["inv_freq"].cpu(), hq,
                                    hkv, d, None if t["qw"] is None else t["qw"].cpu(),
                                    None if t["kw"] is None else t["kw"].cpu(), eps, inter, factor)
    want_k, want_v = t["k"].cpu().double().view(-1, hkv, d), t["v"].cpu().clone().view(-1, hkv, d)
    mag_k = torch.zeros_like(want_k)
    written = torch.zeros(want_k.shape[0], dtype=torch.bool)
    before_k = t["k"].cpu().view(-1, hkv, d).clone()
    for i, slot in enumerate(t["slots"].tolist()):
        if i in skipped:
            continue
        want_k[slot], mag_k[slot], want_v[slot], written[slot] = k[i], km[i], v[i], True
    got = qk_norm_rope_write(t["qkv"] if qkv is None else qkv, t["positions"], t["inv_freq"],
                             t["k"], t["v"], t["slots"], hq, q_weight=t["qw"], k_weight=t["kw"],
                             eps=eps, interleaved=inter, attention_factor=factor, out=out)
    half, tiny = torch.finfo(dtype).eps / 2, torch.finfo(dtype).tiny
    err = (got.cpu().double() - q).abs() - (half * q.abs().clamp(min=tiny) + 2.0 ** -19 * qm)
    assert (err <= 0).all(), f"q: {err.max()} past its bound"
    got_k = t["k"].cpu().view(-1, hkv, d)
    assert torch.equal(got_k[~written], before_k[~written])
    err = (got_k.double() - want_k).abs() - (half * want_k.abs().clamp(min=tiny) + 2.0 ** -19 * mag_k)
    assert (err[written] <= 0).all(), f"k: {err[written].max()} past its bound"
    assert torch.equal(t["v"].cpu().view(-1, hkv, d), want_v)
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("tokens,hq,hkv,d,rot", [
    (1, 14, 2, 64, 64), (5, 28, 4, 128, 128), (33, 8, 2, 96, 64), (7, 4, 2, 16, 8),
    (3, 10, 2, 80, 40), (1100, 6, 3, 32, 32), (2, 16, 1, 128, 64), (3, 4, 4, 256, 128),
    (9, 3, 1, 10, 6), (2, 2, 1, 24, 2), (1030, 2, 1, 72, 12)])
def test_formula(device, dtype, inter, tokens, hq, hkv, d, rot):
    t = make(device, tokens, hq, hkv, d, rot, dtype, seed=tokens + d)
    check(t, hq, hkv, d, inter=inter)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("inter", [False, True])
def test_without_norm_and_with_a_factor(device, dtype, inter):
    t = make(device, 40, 14, 2, 64, 48, dtype, seed=3, norm=False, i32=True)
    check(t, 14, 2, 64, inter=inter, factor=1.25)


def test_far_positions(device):
    t = make(device, 64, 4, 2, 64, 64, torch.float32, seed=4, far=10 ** 9)
    t["positions"][:3] = torch.tensor([0, 2 ** 40 + 1, 10 ** 9 - 1], device=device)
    # At 2^40 the reference's own product in 64 bits is off by 2^-13 radians.
    keep = torch.ones(64, dtype=torch.bool)
    keep[1] = False
    (q, qm), _, _ = reference(t["qkv"].cpu(), t["positions"].cpu(), t["inv_freq"].cpu(), 4, 2, 64,
                              t["qw"].cpu(), t["kw"].cpu(), 1e-6, False, 1.0)
    got = qk_norm_rope_write(t["qkv"], t["positions"], t["inv_freq"], t["k"], t["v"], t["slots"],
                             4, q_weight=t["qw"], k_weight=t["kw"]).cpu().double()
    # The reference's product of 1e9 and the frequency is off by 2^-24.
    err = (got - q).abs() - (2.0 ** -24 * q.abs() + 2.0 ** -18 * qm)
    assert (err[keep] <= 0).all()
    assert (got[1] - q[1]).abs().max() <= 2.0 ** -12 * qm[1].max()


@pytest.mark.parametrize("norm", [False, True])
def test_slots_outside_the_cache_write_nothing(device, norm):
    t = make(device, 9, 6, 2, 64, 64, torch.bfloat16, seed=5, norm=norm)
    slots = t["slots"]
    slots[2], slots[5], slots[7] = -1, t["k"].shape[0] * BS, 2 ** 40
    check(t, 6, 2, 64, skipped=(2, 5, 7))


def test_strided_rows_and_out(device):
    t = make(device, 21, 6, 2, 64, 32, torch.float16, seed=6)
    wide = torch.zeros(21, 10 * 64 + 24, dtype=torch.float16, device=device)
    rows = wide[:, 8:8 + 640]
    rows.copy_(t["qkv"])
    # Rows at 2-byte alignment fall back to single elements.
    odd = torch.zeros(21 * 641 + 1, dtype=torch.float16, device=device)[1:].view(21, 641)[:, :640]
    odd.copy_(t["qkv"])
    big = torch.full((21, 8, 64), 7.0, dtype=torch.float16, device=device)
    first = check(t, 6, 2, 64, qkv=rows, out=big[:, 1:7])
    assert (big[:, 0] == 7).all() and (big[:, 7] == 7).all()
    second = check(t, 6, 2, 64, qkv=odd)
    assert torch.equal(first, second)
    third = check(t, 6, 2, 64)
    assert torch.equal(first, third)


def test_values_that_are_not_finite_stay_in_their_head(device):
    t = make(device, 4, 4, 2, 64, 32, torch.float32, seed=7, norm=False)
    t["qkv"][1, 64 + 40] = math.inf  # head 1, past the rotated part
    t["qkv"][2, 3] = math.nan        # head 0, pair (3, 19)
    got = qk_norm_rope_write(t["qkv"], t["positions"], t["inv_freq"], t["k"], t["v"], t["slots"], 4)
    bad = ~torch.isfinite(got)
    want = torch.zeros_like(bad)
    want[1, 1, 40] = want[2, 0, 3] = want[2, 0, 19] = True
    assert torch.equal(bad, want)


def test_empty_call_and_model_dtype_frequencies(device):
    t = make(device, 3, 4, 2, 16, 16, torch.bfloat16, seed=8)
    out = qk_norm_rope_write(t["qkv"][:0], t["positions"][:0], t["inv_freq"], t["k"], t["v"],
                             t["slots"][:0], 4)
    assert out.shape == (0, 4, 16)
    t["inv_freq"] = t["inv_freq"].bfloat16()
    check(t, 4, 2, 16)


def test_captured_and_replayed(device):
    t = make(device, 17, 14, 2, 64, 64, torch.bfloat16, seed=9)

    def call(x):
        return qk_norm_rope_write(x, t["positions"], t["inv_freq"], t["k"], t["v"], t["slots"], 14,
                                  q_weight=t["qw"], k_weight=t["kw"])

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        call(t["qkv"])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    static = t["qkv"].clone()
    with torch.cuda.graph(graph):
        out = call(static)
    for i in range(3):
        static.copy_(t["qkv"] * (i + 1))
        graph.replay()
        torch.cuda.synchronize()
        k1, v1 = t["k"].clone(), t["v"].clone()
        want = call(static)
        assert torch.equal(out, want) and torch.equal(k1, t["k"]) and torch.equal(v1, t["v"])


def test_other_stream(device):
    t = make(device, 300, 8, 2, 128, 128, torch.bfloat16, seed=10)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        check(t, 8, 2, 128)
    torch.cuda.current_stream().wait_stream(side)
