"""What the drafted-tree, key-eviction and sparse-attention calls refuse, in Python and at the C
ABI, and their sizes at their ends. Nothing here reaches a GPU: the operands are CPU
tensors or numbers that are never dereferenced."""

from __future__ import annotations

import math

import pytest
import torch

from mini_llm_runtime_amd import _lib
from mini_llm_runtime_amd.kernels import key_eviction, sparse_attention, tree_attention

BS = 16
BF = torch.bfloat16


def cache(d=16, dtype=BF, hkv=2, blocks=4):
    return torch.zeros(blocks, BS, hkv, d, dtype=dtype)


def attention_args(**change):
    a = dict(q=torch.zeros(3, 4, 16, dtype=BF), k_cache=cache(), v_cache=cache(), block_size=BS)
    a.update(change)
    return a


ATTENTION = [
    (dict(q=torch.zeros(3, 64)), ValueError, "q must have shape"),
    (dict(k_cache=torch.zeros(4, BS, 16)), ValueError, "k_cache and v_cache must have shape"),
    (dict(v_cache=torch.zeros(3, BS, 2, 16)), ValueError, "same shape"),
    (dict(q=torch.zeros(3, 4, 32, dtype=BF)), ValueError, "same head_dim"),
    (dict(q=torch.zeros(3, 3, 16, dtype=BF)), ValueError, "divisible"),
    (dict(block_size=8), ValueError, "block_size"),
    (dict(q=torch.zeros(3, 4, 16)), TypeError, "one dtype"),
    (dict(q=torch.zeros(3, 4, 16, dtype=torch.float64)), TypeError, "unsupported dtype"),
    (dict(softcap=-1.0), ValueError, "softcap"),
    (dict(softcap=math.nan), ValueError, "softcap"),
    (dict(softcap=1e-31), ValueError, "softcap"),
    (dict(), RuntimeError, "HIP devices"),
] + [(dict(q=torch.zeros(3, 4, d, dtype=t), k_cache=cache(d, t), v_cache=cache(d, t)), ValueError,
      "head_dim in multiples") for d, t in ((12, BF), (136, torch.float16), (6, torch.float32))]


@pytest.mark.parametrize("change,error,needle", ATTENTION)
def test_attention_calls(change, error, needle):
    a = attention_args(**change)
    bt, three = torch.zeros(3, 2, dtype=torch.long), torch.tensor([1, 2, 3])
    with pytest.raises(error, match=needle):
        tree_attention.paged_attention_tree(
            **a, block_tables=bt, query_start_loc=torch.arange(4), context_lens=three,
            ancestors=torch.ones(3, 1, dtype=torch.long))
    with pytest.raises(error, match=needle):
        key_eviction.paged_attention_decode_weighted(
            **a, key_weights=torch.zeros(4, 2, BS), block_tables=bt, seq_lens=three)
    with pytest.raises(error, match=needle):
        sparse_attention.paged_attention_decode_sparse(
            **a, key_bounds=torch.zeros(4, 2, 2, 16, dtype=BF), block_tables=bt, seq_lens=three,
            budget=4)


@pytest.mark.parametrize("parents,max_nodes,error,needle", [
    (torch.zeros(2, 2, dtype=torch.long), 4, ValueError, "parents"),
    (torch.zeros(2, dtype=torch.long), 0, ValueError, "max_nodes"),
    (torch.zeros(2, dtype=torch.long), -64, ValueError, "max_nodes"),
    (torch.zeros(2, dtype=torch.long), 4097, ValueError, "max_nodes"),
    (torch.zeros(2, dtype=torch.long), 4, RuntimeError, "HIP devices")])
def test_tree_ancestors(parents, max_nodes, error, needle):
    with pytest.raises(error, match=needle):
        tree_attention.tree_ancestors(parents, torch.tensor([0, 2]), max_nodes)


@pytest.mark.parametrize("lens,words,fits", [
    ([], 1, True), ([64, 0, 64], 1, True), ([64, 65], 1, False), ([65, 128], 2, True),
    ([129], 2, False)])
def test_tree_words(lens, words, fits):
    """Sequences are held against the words, whatever a caller gave as the most of them."""
    qsl = torch.tensor([0, *lens]).cumsum(0)
    if fits:
        tree_attention._validate_words(qsl, words)
    else:
        with pytest.raises(ValueError, match="a bit for every drafted token"):
            tree_attention._validate_words(qsl, words)


def cache_args(**change):
    a = dict(k_cache=cache(), v_cache=cache(), block_size=BS)
    a.update(change)
    return a


@pytest.mark.parametrize("change,error,needle", [
    (dict(k_cache=torch.zeros(4, BS, 16)), ValueError, "k_cache and v_cache must have shape"),
    (dict(v_cache=cache(32)), ValueError, "same shape"),
    (dict(block_size=8), ValueError, "block_size"),
    (dict(k_cache=cache(dtype=torch.float64)), TypeError, "unsupported dtype"),
    (dict(v_cache=cache(dtype=torch.float16)), TypeError, "one dtype"),
    (dict(k_cache=cache(12), v_cache=cache(12)), ValueError, "head_dim in multiples"),
    (dict(k_cache=cache(1032), v_cache=cache(1032)), ValueError, "head_dim in multiples"),
    (dict(k_cache=cache(32)[..., :16]), ValueError, "contiguous"),
    (dict(), RuntimeError, "HIP devices")])
def test_moves(change, error, needle):
    a, bt = cache_args(**change), torch.zeros(1, 2, dtype=torch.long)
    with pytest.raises(error, match=needle):
        key_eviction.compact_keys(**a, block_tables=bt, kept=torch.zeros(1, 2, dtype=torch.long))
    with pytest.raises(error, match=needle):
        key_eviction.evict_keys(**a, key_weights=torch.zeros(4, 2, BS), block_tables=bt,
                                seq_lens=torch.tensor([3]), budget=8)


@pytest.mark.parametrize("weights", [
    torch.zeros(4, BS, 2), torch.zeros(3, 2, BS), torch.zeros(4, 2, BS, dtype=BF),
    torch.zeros(4, BS, 2).transpose(1, 2), torch.zeros(1, 2, BS).expand(4, 2, BS)])
def test_key_weights(weights):
    with pytest.raises(ValueError, match="key_weights"):
        key_eviction._check_weights(weights, cache())


@pytest.mark.parametrize("bounds", [
    torch.zeros(4, 2, 2, 8, dtype=BF), torch.zeros(4, 2, 2, 16), torch.zeros(4, 2, 16, dtype=BF),
    torch.zeros(4, 2, 2, 32, dtype=BF)[..., :16]])
def test_key_bounds(bounds):
    with pytest.raises(ValueError, match="key_bounds"):
        sparse_attention._check_bounds(bounds, cache())
    with pytest.raises(ValueError, match="key_bounds"):
        sparse_attention.update_key_bounds(cache(), bounds, torch.zeros(1, 2, dtype=torch.long),
                                           torch.tensor([3]), BS)


@pytest.mark.parametrize("change,error,needle", [
    (dict(k_cache=torch.zeros(4, BS, 16)), ValueError, "k_cache must have shape"),
    (dict(block_size=8), ValueError, "block_size"),
    (dict(k_cache=cache(dtype=torch.float64)), TypeError, "unsupported dtype"),
    (dict(k_cache=cache(12)), ValueError, "head_dim in multiples"),
    (dict(k_cache=cache(32)[..., :16]), ValueError, "contiguous"),
    (dict(), RuntimeError, "HIP devices")])
def test_update_key_bounds(change, error, needle):
    a = dict(k_cache=cache(), block_size=BS)
    a.update(change)
    with pytest.raises(error, match=needle):
        sparse_attention.update_key_bounds(
            **a, key_bounds=torch.zeros(4, 2, 2, 16, dtype=BF),
            block_tables=torch.zeros(1, 2, dtype=torch.long), seq_lens=torch.tensor([3]))


@pytest.mark.parametrize("kept,start,needle", [
    ([[[3, 2]]], None, "ascend"), ([[[2, 2]]], None, "ascend"), ([[[-1, 3]]], None, "ascend"),
    ([[[5, -1, 6]]], None, "ascend"), ([[[0, 1]]], [1], "at least start"),
    ([[[20, 31]]], [-1], "negative"), ([[[31, 32]]], None, "enough blocks"),
    ([[[1 << 40]]], None, "enough blocks")])
def test_lists(kept, start, needle):
    table = torch.tensor([[2, 1]])
    with pytest.raises(ValueError, match=needle):
        key_eviction._validate_lists(table, torch.tensor(kept),
                                     None if start is None else torch.tensor(start), BS, 4)


def test_lists_and_their_blocks():
    lists = torch.tensor([[[17, 20]], [[-1, -1]]])

    def check(table, start=None, kept=lists):
        key_eviction._validate_lists(torch.tensor(table), kept,
                                     None if start is None else torch.tensor(start), BS, 4)

    check([[2, 1], [2, 1]])  # the second moves nothing
    check([[-1, 1], [9, 9]], [16, 0])  # blocks before the start are not touched
    both = torch.tensor([[[17, 20]], [[16, 31]]])
    check([[0, 1], [0, 2]], [16, 16], both)
    for table, start, needle in (([[0, 1], [0, 2]], [0, 16], None), ([[0, 1], [3, 1]], [16, 16], 1),
                                 ([[0, 1], [0, 2]], [0, 0], 1), ([[1, 1], [0, 2]], [0, 16], 1)):
        if needle is None:
            check(table, start, both)
            continue
        with pytest.raises(ValueError, match="share a block"):
            check(table, start, both)
    for table in ([[-1, 1], [2, 3]], [[0, 4], [2, 3]], [[0, 1 << 40], [2, 3]]):
        with pytest.raises(ValueError, match="physical block"):
            check(table, None, both)


@pytest.mark.parametrize("tables,lens,shared", [
    ([[0, 1], [0, 2]], [20, 32], False),          # a whole first block in common
    ([[0, 1], [0, 2]], [20, 16], True),           # whose last key is the second's newest
    ([[0, 1], [0, 1]], [20, 20], True),           # the same keys throughout
    ([[0, 1], [0, 1]], [20, 24], True),           # the first's newest is a key of the second
    ([[0, 1], [2, 0]], [17, 18], True),           # at another place there
    ([[0, 1], [2, 0]], [16, 17], True),
    ([[0, 0]], [18], True),                       # twice in one request
    ([[0, 1], [1, 0]], [16, 16], False),          # columns past the end are not used
    ([[0, -1], [1, -1], [2, 0]], [1, 16, 16], False),
    ([[3, 1], [3, 2], [3, 0]], [17, 18, 19], False), ([[2]], [1], False)])
def test_newest_keys(tables, lens, shared):
    got = key_eviction._newest_is_shared(torch.tensor(tables), torch.tensor(lens), BS)
    assert bool(got) == shared


def test_newest_keys_against_all_pairs():
    """Random tables over few blocks, against a count of the requests that hold each key."""
    gen, seen = torch.Generator().manual_seed(1), set()
    for case in range(300):
        bs, batch, width = 1 + case % 3, 1 + case % 4, 3
        tables = torch.randint(0, 9, (batch, width), generator=gen)
        lens = torch.randint(1, width * bs + 1, (batch,), generator=gen)
        held = [(tables[b, i // bs].item(), i % bs) for b in range(batch) for i in range(lens[b])]
        newest = [(tables[b, (lens[b] - 1) // bs].item(), ((lens[b] - 1) % bs).item())
                  for b in range(batch)]
        want = any(held.count(key) > 1 for key in newest)
        assert bool(key_eviction._newest_is_shared(tables, lens, bs)) == want
        seen.add(want)
    assert seen == {True, False}


P = 1 << 20  # a pointer that is aligned and never read


def attention_abi(**change):
    a = dict(q=P, qb=64, qh=16, k=P, v=P, nb=4, bs=BS, hkv=2, d=16, bt=P, bst=2, width=2, lens=P,
             hq=4, scale=0.25, cap=0.0, dtype=2, ws=P, nbytes=1 << 40, out=P, ob=64, oh=16)
    a.update(change)
    return a


def tree_abi(a, **more):
    m = dict(qsl=P, bits=P, words=1, seqs=3, total=9, longest=5)
    m.update(more)
    return _lib.load().mlr_paged_attention_tree(
        a["q"], a["qb"], a["qh"], a["k"], a["v"], a["nb"], a["bs"], a["hkv"], a["d"], a["bt"],
        a["bst"], a["width"], m["qsl"], a["lens"], m["bits"], m["words"], m["seqs"], m["total"],
        m["longest"], a["hq"], a["scale"], a["cap"], a["dtype"], a["ws"], a["nbytes"], a["out"],
        a["ob"], a["oh"], None)


def weigh_abi(a, weights=P, batch=3):
    return _lib.load().mlr_paged_decode_weighted(
        a["q"], a["qb"], a["qh"], a["k"], a["v"], weights, a["nb"], a["bs"], a["hkv"], a["d"],
        a["bt"], a["bst"], a["width"], a["lens"], batch, a["hq"], a["scale"], a["cap"], a["dtype"],
        a["ws"], a["nbytes"], a["out"], a["ob"], a["oh"], None)


def sparse_abi(a, bounds=P, batch=3, budget=8, sinks=1, recent=1):
    return _lib.load().mlr_paged_decode_sparse(
        a["q"], a["qb"], a["qh"], a["k"], a["v"], bounds, a["nb"], a["bs"], a["hkv"], a["d"],
        a["bt"], a["bst"], a["width"], a["lens"], batch, a["hq"], budget, sinks, recent,
        a["scale"], a["cap"], a["dtype"], None, a["ws"], a["nbytes"], a["out"], a["ob"], a["oh"],
        None)


@pytest.mark.parametrize("call", [tree_abi, weigh_abi, sparse_abi])
@pytest.mark.parametrize("change,needle", [
    (dict(dtype=3), b"dtype"), (dict(hq=3), b"multiple"), (dict(hkv=0), b"multiple"),
    (dict(d=20), b"head_dim"), (dict(d=136), b"head_dim"), (dict(nb=0), b"blocks"),
    (dict(bs=0), b"blocks"), (dict(width=1 << 31), b"2^31 positions"), (dict(cap=-1.0), b"softcap"),
    (dict(cap=math.nan), b"softcap"), (dict(scale=math.inf), b"scale"), (dict(qb=60), b"16 bytes"),
    (dict(q=P + 2), b"16 bytes"), (dict(k=P + 8), b"aligned"), (dict(lens=None), b"null"),
    (dict(bt=None), b"null"), (dict(out=None), b"null"),
    (dict(width=1000, ws=None, nbytes=0), b"workspace"), (dict(width=1000, nbytes=64), b"workspace")])
def test_attention_abi(call, change, needle):
    assert call(attention_abi(**change)) == 1 and needle in _lib.load().mlr_last_error()


def test_own_arguments_abi():
    lib, a = _lib.load(), attention_abi()
    for more, needle in [
            (dict(qsl=None), b"null"), (dict(bits=None), b"null"), (dict(words=0), b"words"),
            (dict(words=-1), b"words"), (dict(total=-1), b"token counts"),
            (dict(longest=1 << 40, total=1 << 40), b"too many query rows")]:
        assert tree_abi(a, **more) == 1 and needle in lib.mlr_last_error(), more
    for more in (dict(total=0), dict(seqs=0), dict(longest=0)):
        assert tree_abi(a, **more) == 0
    assert weigh_abi(a, batch=-1) == 1 and b"sequences" in lib.mlr_last_error()
    assert weigh_abi(a, weights=None) == 1 and b"null" in lib.mlr_last_error()
    assert weigh_abi(a, batch=0) == 0 and sparse_abi(a, batch=0) == 0
    for more, needle in [(dict(bounds=None), b"null"), (dict(bounds=P + 8), b"aligned"),
                         (dict(batch=-1), b"sequences"), (dict(budget=0), b"budget"),
                         (dict(recent=0), b"budget"), (dict(sinks=-1), b"budget"),
                         (dict(sinks=8), b"budget"), (dict(budget=1 << 31), b"budget"),
                         (dict(sinks=(1 << 63) - 1, recent=8), b"budget")]:
        assert sparse_abi(a, **more) == 1 and needle in lib.mlr_last_error(), more


def evict_abi(**change):
    a = dict(k=P, v=P, w=P, nb=4, bs=BS, hkv=2, d=16, bt=P, bst=2, width=2, lens=P, batch=3, budget=8,
             sinks=1, recent=1, dtype=2, kept=P, new=P, stream=None)
    a.update(change)
    return _lib.load().mlr_evict_keys(*a.values())


def compact_abi(**change):
    a = dict(k=P, v=P, w=None, nb=4, bs=BS, hkv=2, d=16, bt=P, bst=2, width=2, kept=P, sb=8, sh=4, n=4,
             start=None, batch=3, dtype=2, stream=None)
    a.update(change)
    return _lib.load().mlr_compact_keys(*a.values())


def bounds_abi(**change):
    a = dict(k=P, b=P, nb=4, bs=BS, hkv=2, d=16, bt=P, bst=2, width=2, lens=P, starts=None, most=4,
             batch=3, dtype=2, stream=None)
    a.update(change)
    return _lib.load().mlr_update_key_bounds(*a.values())


@pytest.mark.parametrize("call", [evict_abi, compact_abi, bounds_abi])
@pytest.mark.parametrize("change,needle", [
    (dict(dtype=3), b"dtype"), (dict(batch=-1), b"sequences"), (dict(batch=1 << 24), b"sequences"),
    (dict(hkv=0), b""), (dict(hkv=1 << 16), b""), (dict(d=0), b"16 bytes"), (dict(d=12), b"16 bytes"),
    (dict(d=1032), b"16 bytes"), (dict(nb=0), b"blocks"), (dict(nb=1 << 31), b"block"),
    (dict(bs=0), b"block"), (dict(width=1 << 27), b"2^31 positions"), (dict(width=-1), b"block"),
    (dict(k=None), b"null"), (dict(bt=None), b"null"), (dict(k=P + 8), b"aligned")])
def test_cache_abi(call, change, needle):
    if call is bounds_abi and change == dict(nb=0):
        needle = b"block"
    assert call(**change) == 1 and needle in _lib.load().mlr_last_error()


def test_lists_abi():
    lib = _lib.load()
    for change, needle in [(dict(budget=-1), b"budget"), (dict(sinks=8), b"budget"),
                           (dict(recent=9), b"budget"), (dict(sinks=-1), b"budget"),
                           (dict(budget=1 << 31), b"budget"), (dict(w=None), b"null"),
                           (dict(lens=None), b"null"), (dict(kept=None), b"null"),
                           (dict(new=None), b"null"), (dict(batch=1 << 23, hkv=64), b"too many lists"),
                           (dict(sinks=(1 << 63) - 1, recent=(1 << 63) - 1), b"budget")]:
        assert evict_abi(**change) == 1 and needle in lib.mlr_last_error(), change
    for change, needle in [(dict(n=-1), b"kept"), (dict(n=1 << 31), b"kept"),
                           (dict(kept=None), b"null"),
                           (dict(batch=1 << 23, hkv=64), b"too many lists")]:
        assert compact_abi(**change) == 1 and needle in lib.mlr_last_error(), change
    assert bounds_abi(most=-1) == 1 and b"max_new" in lib.mlr_last_error()
    assert bounds_abi(b=None) == 1 and b"null" in lib.mlr_last_error()
    assert evict_abi(batch=0) == 0 and compact_abi(batch=0) == 0 and compact_abi(n=0) == 0
    assert bounds_abi(batch=0) == 0 and bounds_abi(width=0, bt=None) == 0
    assert bounds_abi(most=0, starts=P) == 0


def test_ancestors_abi():
    lib = _lib.load()

    def ancestors(**change):
        a = dict(parents=P, qsl=P, seqs=3, total=9, words=1, out=P, stream=None)
        a.update(change)
        return lib.mlr_tree_ancestors(*a.values())

    for change in (dict(parents=None), dict(qsl=None), dict(out=None), dict(seqs=-1),
                   dict(seqs=1 << 24), dict(total=-1), dict(words=0), dict(words=65)):
        assert ancestors(**change) == 1 and b"mlr_tree_ancestors" in lib.mlr_last_error(), change
    assert ancestors(seqs=0) == 0 and ancestors(total=0) == 0


MB = 1 << 20


@pytest.mark.parametrize("dtype", [torch.float32, BF])
@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (32, 8, 128)])
def test_workspaces(dtype, hq, hkv, d):
    """Some hundred MB at most but for the scores of a weighing decode, which have 4 bytes
    for every head and covered position."""
    lib, code = _lib.load(), _lib.DTYPE_CODES[dtype]
    for seqs in (1, 16, 64, 1000):
        for longest in (1, 16, 64, 500):
            tree = lib.mlr_paged_attention_tree_workspace_size(seqs, longest, 2048, BS, hq, hkv, d,
                                                               code)
            assert tree <= 512 * MB
        scores = 4 * seqs * hq * 2048 * BS
        weigh = lib.mlr_paged_decode_weighted_workspace_size(seqs, hq, hkv, d, 2048 * BS)
        assert scores <= weigh <= scores + 256 * MB
        sparse = lib.mlr_paged_decode_sparse_workspace_size(seqs, hq, hkv, d, 2048, BS, 256, code)
        keys = 8 * seqs * hkv * (2 * 2048 + 256)
        assert 0 < sparse <= keys + 256 * MB
    assert lib.mlr_paged_attention_tree_workspace_size(0, 5, 8, BS, hq, hkv, d, code) == 0
    assert lib.mlr_paged_decode_weighted_workspace_size(3, hq, hkv, d, 0) == 0
    assert lib.mlr_paged_decode_sparse_workspace_size(3, hq, hkv, d, 0, BS, 8, code) == 0
