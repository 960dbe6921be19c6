"""Key bounds and sparse decode against 64 bits."""

from __future__ import annotations

import pytest
import torch

from mini_llm_runtime_amd.kernels.scored_attention import paged_attention_decode_scored
from mini_llm_runtime_amd.kernels.sparse_attention import (paged_attention_decode_sparse,
                                                           update_key_bounds)

import selection_oracle as so

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def bounds_of(k, tables, lens, starts, bs, before):
    out = before.clone()
    for i, n in enumerate(lens):
        first = 0 if starts is None else starts[i] // bs
        if starts is not None and starts[i] >= n:
            continue
        for j in range(first, -(-n // bs)):
            keys = k[tables[i, j], :min(bs, n - j * bs)]
            out[tables[i, j], 0], out[tables[i, j], 1] = keys.amin(0), keys.amax(0)
    return out


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("heads", [(2, 64), (1, 128), (3, 8), (4, 80), (2, 256)])
@pytest.mark.parametrize("block_size", [16, 1, 7, 64])
def test_bounds(device, dtype, heads, block_size):
    lens = [1, 15, 16, 17, 200]
    k, _, tables = so.pool(lens, block_size, *heads, dtype, 3)
    before = torch.full((k.shape[0], 2, *heads), 3.0).to(dtype)
    for starts, new in ((None, None), ([0, 14, 15, 16, 199], 1), ([1, 3, 0, 17, 150], 50),
                        ([0, 14, 15, 16, 199], None)):
        got = before.to(device)
        update_key_bounds(k.to(device), got, tables.to(device), torch.tensor(lens).to(device),
                          block_size,
                          starts=None if starts is None else torch.tensor(starts).to(device),
                          max_new=new)
        assert torch.equal(got.cpu(), bounds_of(k, tables, lens, starts, block_size, before))


@pytest.mark.parametrize("most", [5, 1 << 40, 1 << 70])
def test_bounds_of_a_range_said_to_be_long(device, most):
    """max_new past what the tables cover, or past 64 bits, is all that they cover; without
    starts it says nothing."""
    lens, starts = [70, 33], [68, 28]
    k, v, tables = so.pool(lens, 16, 2, 64, BF, 0)
    before = torch.zeros(k.shape[0], 2, 2, 64, dtype=BF)
    for first in (starts, None):
        got = before.to(device)
        update_key_bounds(k.to(device), got, tables.to(device), torch.tensor(lens).to(device), 16,
                          starts=None if first is None else torch.tensor(first).to(device),
                          max_new=most if first else 0)
        assert torch.equal(got.cpu(), bounds_of(k, tables, lens, first, 16, before.clone()))


@pytest.mark.parametrize("dtype", [BF, FP, F32])
def test_bounds_of_odd_values(device, dtype):
    """A NaN stays, infinities bound, and what lies behind the last key is not read."""
    k, _, tables = so.pool([40], 16, 2, 64, dtype, 3)
    k[tables[0, 0], 3, 0, 5] = float("nan")
    k[tables[0, 1], 2, 1, 7] = float("inf")
    k[tables[0, 1], 9, 1, 7] = -float("inf")
    k[tables[0, 2], 8:] = float("nan")
    got = torch.zeros(k.shape[0], 2, 2, 64, dtype=dtype, device=device)
    update_key_bounds(k.to(device), got, tables.to(device), torch.tensor([40]).to(device), 16)
    want = bounds_of(k, tables, [40], None, 16, torch.zeros(k.shape[0], 2, 2, 64, dtype=dtype))
    torch.testing.assert_close(got.cpu(), want, rtol=0, atol=0, equal_nan=True)
    assert want[tables[0, 0], :, 0, 5].isnan().all()
    assert want[tables[0, 2]].isfinite().all()


def test_bounds_padded_rows_and_bad_blocks(device):
    k, _, tables = so.pool([40, 40], 16, 2, 64, BF, 3)
    want = bounds_of(k, tables[1:], [40], None, 16, torch.zeros(k.shape[0], 2, 2, 64, dtype=BF))
    want[tables[1, 1]] = 0
    tables[1, 1] = 1 << 33
    got = torch.zeros(k.shape[0], 2, 2, 64, dtype=BF, device=device)
    update_key_bounds(k.to(device), got, tables.to(device), torch.tensor([0, 40]).to(device), 16,
                      validate=False)
    assert torch.equal(got.cpu(), want)


MANY = 4096  # blocks of a table


def run_case(device, dtype, heads, lens, budget, sinks=1, recent=1, block_size=16, cap=0.0,
             scale=None, seed=0, validate=True, change=None, width=None):
    hq, hkv, d = heads
    if width == MANY:  # scores in 32 bits first, which a few lists are not worth
        lens = lens + [1] * (-(-(6 << 20) // (MANY * hkv * d)) - len(lens))
    k, v, tables = so.pool(lens, block_size, hkv, d, dtype, seed, width=width)
    gen = torch.Generator().manual_seed(seed + 1)
    q = torch.randn(len(lens), hq, d, generator=gen).to(dtype)
    bounds = torch.zeros(k.shape[0], 2, hkv, d, dtype=dtype)
    bounds = bounds_of(k, tables, lens, None, block_size, bounds)
    if change is not None:
        change(q, k, v, bounds, tables)
    scale = d ** -0.5 if scale is None else scale
    got, blocks = paged_attention_decode_sparse(
        q.to(device), k.to(device), v.to(device), bounds.to(device), tables.to(device),
        torch.tensor(lens).to(device), block_size, budget, sinks=sinks, recent=recent,
        softcap=cap, scale=scale, return_blocks=True, validate=validate)
    for i, n in enumerate(lens):
        count = -(-n // block_size)
        used = tables[i, :count].clamp(0, k.shape[0] - 1)
        x = -q[i] if scale < 0 else q[i]
        score = so.block_scores(x, bounds[used, 0], bounds[used, 1])
        seen = torch.zeros(1, hkv, n, dtype=torch.bool)
        for h in range(hkv):
            stay = so.choose(score[h], sinks, recent, budget)
            assert blocks[i, h].tolist() == stay + [-1] * (budget - len(stay)), (i, h)
            for j in stay:
                seen[0, h, j * block_size:(j + 1) * block_size] = True
        slot = so.slots(tables[i], n, block_size).clamp(min=0)
        want, bound, _, _ = so.attend(q[i:i + 1], k.view(-1, hkv, d)[slot],
                                      v.view(-1, hkv, d)[slot], seen, scale, cap, dtype)
        so.assert_within(got[i:i + 1], want, bound, f"request {i}")
    return got, blocks


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("heads", [(14, 2, 64), (8, 2, 128), (4, 4, 96), (6, 2, 40), (16, 1, 16),
                                   (80, 1, 32), (3, 1, 8)])
def test_sparse(device, dtype, heads):
    run_case(device, dtype, heads, [1, 16, 17, 100, 500, 513], 8, sinks=1, recent=2)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("block_size", [1, 5, 8, 32, 24])
def test_block_sizes(device, dtype, block_size):
    run_case(device, dtype, (4, 2, 64), [1, 31, 330], 6, block_size=block_size)


@pytest.mark.parametrize("budget,sinks,recent", [(1, 0, 1), (2, 1, 1), (5, 0, 5), (5, 4, 1),
                                                 (9, 0, 1), (100, 3, 3)])
def test_budgets(device, budget, sinks, recent):
    run_case(device, BF, (14, 2, 64), [1, 80, 81, 400, 1000], budget, sinks, recent)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("heads", [(14, 2, 64), (8, 2, 128), (4, 4, 96), (6, 2, 40), (40, 1, 16),
                                   (80, 1, 32), (3, 1, 8)])
def test_many_lists_of_long_tables(device, dtype, heads):
    for budget, sinks, recent in ((8, 1, 2), (3, 0, 3), (40, 4, 1), (400, 0, 1)):
        run_case(device, dtype, heads, [1, 16, 17, 1000, 5000, 5001, 65536], budget, sinks, recent,
                 width=MANY)
    run_case(device, dtype, heads, [3000, 200], 5, cap=10.0, scale=-0.1, width=MANY)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_long_contexts(device, dtype):
    run_case(device, dtype, (4, 2, 64), [20000, 7], 100, recent=3)
    run_case(device, dtype, (2, 2, 8), [150000], 700, recent=3)


@pytest.mark.parametrize("dtype", [BF, FP, F32])
def test_capped_and_negative_scale(device, dtype):
    run_case(device, dtype, (14, 2, 64), [300, 200], 5, cap=10.0)
    run_case(device, dtype, (14, 2, 64), [300, 200], 5, scale=-0.1)


# Up to 128 blocks a table's scores and choice are one launch, past that two, and with many
# lists of long tables 16-bit scores are made in 32 bits first.
WIDTHS = pytest.mark.parametrize("width", [None, 300, MANY])


@WIDTHS
@pytest.mark.parametrize("dtype", [BF, F32])
def test_ties_go_to_the_lower_block(device, dtype, width):
    def change(q, k, v, bounds, tables):
        bounds[:, 0] = -1.0
        bounds[:, 1] = 1.0
        bounds[tables[0, 20], 1] = 2.0

    _, blocks = run_case(device, dtype, (14, 2, 64), [600], 6, change=change, width=width)
    assert blocks[0, 0].tolist() == [0, 1, 2, 3, 20, 37]


@WIDTHS
@pytest.mark.parametrize("dtype", [BF, FP, F32])
def test_scores_apart_by_less_than_32_bits_hold(device, dtype, width):
    """Sums of terms of unlike size, whose 32-bit sums would be equal."""
    def change(q, k, v, bounds, tables):
        q[:] = 1.0
        q[0, :, 1] = 2.0 ** -10
        bounds[:] = 1.0
        bounds[:, :, :, 0] = 2.0 ** 14
        for j in (9, 5, 30):
            bounds[tables[0, j], 1, :, 1] = 1.0 + 2.0 ** -7

    _, blocks = run_case(device, dtype, (2, 1, 64), [600], 5, change=change, width=width)
    assert blocks[0, 0].tolist() == [0, 5, 9, 30, 37]


@WIDTHS
@pytest.mark.parametrize("dtype", [BF, FP, F32])
def test_bounds_that_are_not_finite(device, dtype, width):
    """A head's NaN does not count, and a block of NaN scores lowest; infinities score."""
    def change(q, k, v, bounds, tables):
        bounds[tables[0, 3]] = float("nan")
        bounds[tables[0, 5], 1, 0, 2] = float("inf")
        bounds[tables[0, 6], 0, 0, 2] = -float("inf")
        q[0, 0, 2] = 0.0

    run_case(device, dtype, (4, 2, 64), [400], 6, change=change, width=width)


@WIDTHS
@pytest.mark.parametrize("dtype", [BF, F32])
def test_hidden_rows_are_not_read(device, dtype, width):
    """Blocks that are not chosen, and rows behind the last key, may hold anything."""
    def change(q, k, v, bounds, tables):
        for j in range(2, 24):
            bounds[tables[0, j]] = 0.0 if j != 7 else bounds[tables[0, j]].abs() + 5
            if j != 7:
                k[tables[0, j]] = float("nan")
                v[tables[0, j]] = float("nan")
        bounds[tables[0, 1]] = 0.0
        bounds[tables[0, 1], 1] = 100.0
        bounds[tables[0, 1], 0] = -100.0
        bounds[tables[0, 7], 0] = -50.0
        bounds[tables[0, 7], 1] = 50.0
        k[tables[0, 24], 9:] = float("nan")
        v[tables[0, 24], 9:] = float("nan")

    got, _ = run_case(device, dtype, (14, 2, 64), [393], 4, change=change, width=width)
    assert got.isfinite().all()


def test_padded_rows_and_wide_tables(device):
    got, blocks = run_case(device, BF, (14, 2, 64), [0, 400, 0], 5, validate=False, width=64)
    assert (got[0] == 0).all() and (got[2] == 0).all() and (blocks[0] == -1).all()


@WIDTHS
def test_bad_blocks_score_lowest_and_are_masked(device, width):
    lens = [160] + ([1] * 15 if width == MANY else [])
    k, v, tables = so.pool(lens, 16, 2, 64, BF, 0, width=width)
    bounds = bounds_of(k, tables, lens, None, 16, torch.zeros(k.shape[0], 2, 2, 64, dtype=BF))
    q = torch.randn(len(lens), 14, 64, generator=torch.Generator().manual_seed(1)).to(BF)
    tables[0, 4] = 1 << 40
    got, blocks = paged_attention_decode_sparse(
        q.to(device), k.to(device), v.to(device), bounds.to(device), tables.to(device),
        torch.tensor(lens).to(device), 16, 9, return_blocks=True, validate=False)
    assert blocks[0].tolist() == [[0, 1, 2, 3, 5, 6, 7, 8, 9]] * 2
    tables[0, 4] = 0
    seen = torch.ones(1, 160, dtype=torch.bool)
    seen[:, 64:80] = False
    slot = so.slots(tables[0], 160, 16)
    want, bound, _, _ = so.attend(q[:1], k.view(-1, 2, 64)[slot], v.view(-1, 2, 64)[slot], seen,
                                  0.125, 0.0, BF)
    so.assert_within(got[:1], want, bound)


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("heads", [(14, 2, 64), (8, 2, 128), (6, 2, 40), (40, 2, 24)])
@pytest.mark.parametrize("left", [1, 40])
def test_scores_that_32_bits_leave_open(device, dtype, heads, left):
    """Groups of blocks that differ in the last place of one bound: some, more than are
    compared one by one, and all of them open in 32 bits."""
    for alike in (3, 50, 90, 400):
        def change(q, k, v, bounds, tables):
            at = tables[0, 10:10 + alike]
            base = bounds[at[0]].clone()
            bounds[at] = base
            gen = torch.Generator().manual_seed(alike)
            place = torch.randint(0, heads[2], (alike,), generator=gen)
            step = 1.0 + torch.finfo(dtype).eps * torch.randint(-1, 2, (alike,), generator=gen)
            for j, b in enumerate(at):
                bounds[b, 1, :, place[j]] *= step[j].to(dtype)

        run_case(device, dtype, heads, [16 * 420], left + 3, sinks=1, recent=2, change=change,
                 width=MANY)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_scores_past_what_32_bits_hold(device, dtype):
    """Products and sums that overflow 32 bits, subnormal operands, and rows of zeros. The
    blocks hold in all of them; with a query of 3e38 and keys past 1.2 the attention's own
    products pass 3.41e38, the largest 32-bit number, and only the blocks are compared."""
    big = 3e38 if dtype == BF else 65504.0
    tiny = torch.finfo(dtype).tiny / 4

    for kind in ("big", "tiny", "zeros", "mixed"):
        def change(q, k, v, bounds, tables):
            if kind == "zeros":
                bounds.zero_()
            elif kind == "tiny":
                bounds.mul_(tiny)
                q.mul_(tiny)
            else:
                bounds[tables[0, 5:200:3], 1, :, 3] = big
                q[:, :, 3] = big if kind == "big" else 1.0

        q_free = dict(scale=1e-9) if kind == "big" else {}
        run_case(device, dtype, (14, 2, 64), [16 * 300], 20, recent=2, change=change, width=MANY,
                 **q_free)


@pytest.mark.parametrize("scale", [1e-19, -1e-19])
def test_sums_that_overflow_on_their_way(device, scale):
    """A block whose best head has products of -3e38 four times, then as many of 3e38, the
    last two steps larger: its score, 4e36, is past those of many others, 5e35 to 2e36 and all
    unlike, though a sum in 32 bits passes -infinity on its way and the block's other
    heads score far less."""
    sign = 1.0 if scale > 0 else -1.0

    def change(q, k, v, bounds, tables):
        q[0, 0] = 0.0
        q[0, 0, :4], q[0, 0, 4:9] = -1e19 * sign, 1e19 * sign
        at = tables[0, 5:200]
        first = torch.tensor(5e16).to(BF).view(torch.int16)
        bounds[at, 1, 0, 8] = (first + torch.arange(len(at), dtype=torch.int16)).view(BF)
        one = tables[0, 100]
        bounds[one, :, 0, :8] = 3e19
        bounds[one, 1, 0, 7] *= 1 + 2.0 ** -6
        bounds[one, 1, 0, 8] = 1.0

    _, blocks = run_case(device, BF, (14, 2, 64), [16 * 300], 20, recent=2, scale=scale,
                         change=change, width=MANY)
    assert 100 in blocks[0, 0].tolist()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("width", [None, 200, MANY])
@pytest.mark.parametrize("left", [1, 5, 8])
def test_ties_beside_a_block_that_is_not_finite(device, dtype, width, left):
    """Every block of the first sixteen stands sixteen places on once more, and one of the
    first has a bound that is not finite: its whole tile still has the scores of the copies, to
    the last bit, so that the lower place goes first."""
    def change(q, k, v, bounds, tables):
        for i in range(4):
            bounds[tables[i, 16:32]] = bounds[tables[i, :16]]
            bounds[tables[i, 3 + i], 1, :, 5] = float("nan")

    run_case(device, dtype, (14, 2, 64), [16 * 33] * 4, left + 1, sinks=0, recent=1, change=change,
             width=width)


@pytest.mark.parametrize("dtype", [BF, FP, F32])
def test_whole_requests_are_the_scored_decode(device, dtype):
    """A budget of all blocks: no bounds are read, and the result is the decode's; both are
    within the bound of the exact one, hence within twice that of each other."""
    lens = [100, 1, 333]
    k, v, tables = so.pool(lens, 16, 2, 64, dtype, 0)
    q = torch.randn(3, 14, 64, generator=torch.Generator().manual_seed(1)).to(dtype)
    bounds = torch.full((k.shape[0], 2, 2, 64), float("nan"), dtype=dtype)
    args = [x.to(device) for x in (q, k, v)]
    rest = (tables.to(device), torch.tensor(lens).to(device), 16)
    got = paged_attention_decode_sparse(*args, bounds.to(device), *rest, 21)
    want = paged_attention_decode_scored(*args, *rest).double().cpu()
    for i, n in enumerate(lens):
        slot = so.slots(tables[i], n, 16)
        _, bound, _, _ = so.attend(q[i:i + 1], k.view(-1, 2, 64)[slot], v.view(-1, 2, 64)[slot],
                                   torch.ones(1, n, dtype=torch.bool), 0.125, 0.0, dtype)
        so.assert_within(got[i:i + 1], want[i:i + 1], 2 * bound)


def test_strides(device):
    """q as a view of packed rows, an out with wide rows, int32 metadata."""
    k, v, tables = so.pool([300, 100], 16, 2, 64, BF, 0)
    wide = torch.randn(2, 18 * 64, generator=torch.Generator().manual_seed(1)).to(BF).to(device)
    q = wide[:, :14 * 64].view(2, 14, 64)
    bounds = torch.stack([k.amin(1), k.amax(1)], 1).to(device)
    k, v, tables = k.to(device), v.to(device), tables.to(device)
    lens = torch.tensor([300, 100]).to(device)
    want = paged_attention_decode_sparse(q.contiguous(), k, v, bounds, tables, lens, 16, 5)
    out = torch.zeros(2, 14, 100, dtype=BF, device=device)
    got = paged_attention_decode_sparse(q, k, v, bounds, tables.int(), lens.int(), 16, 5,
                                        out=out[..., :64])
    torch.testing.assert_close(got, want, rtol=0, atol=0)
    assert (out[..., 64:] == 0).all()
