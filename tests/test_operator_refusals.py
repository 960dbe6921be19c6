"""What qk_norm_rope_write, the scored attention calls, sample_tokens and
random_sample refuse, in Python and at the C ABI. Nothing here reaches a GPU: the
operands are CPU tensors or numbers that are never dereferenced."""

from __future__ import annotations

import math

import pytest
import torch

from mini_llm_runtime_amd import _lib
from mini_llm_runtime_amd.kernels import pre_attention, sampling, scored_attention
from mini_llm_runtime_amd.runtime import model_runner

BS = 16


def rope_args(**change):
    a = dict(qkv=torch.zeros(3, (4 + 4) * 16, dtype=torch.bfloat16),
             positions=torch.zeros(3, dtype=torch.long), inv_freq=torch.ones(8),
             k_cache=torch.zeros(2, BS, 2, 16, dtype=torch.bfloat16),
             v_cache=torch.zeros(2, BS, 2, 16, dtype=torch.bfloat16),
             slot_mapping=torch.arange(3), num_q_heads=4)
    a.update(change)
    return a


W = torch.ones(16, dtype=torch.bfloat16)


@pytest.mark.parametrize("change,error,needle", [
    (dict(k_cache=torch.zeros(2, BS, 16)), ValueError, "k_cache and v_cache"),
    (dict(num_q_heads=3), ValueError, "multiple of the cache's KV heads"),
    (dict(num_q_heads=0), ValueError, "multiple of the cache's KV heads"),
    (dict(qkv=torch.zeros(3, 100, dtype=torch.bfloat16)), ValueError, "qkv must have shape"),
    (dict(qkv=torch.zeros(3, 128, dtype=torch.float64)), TypeError, "not supported"),
    (dict(qkv=torch.zeros(3, 128)), TypeError, "KV cache dtype"),
    (dict(qkv=torch.zeros(128, 3, dtype=torch.bfloat16).T), ValueError, "contiguous"),
    (dict(qkv=torch.zeros(1, 128, dtype=torch.bfloat16).expand(3, 128)), ValueError, "contiguous"),
    (dict(positions=torch.zeros(3, dtype=torch.int32)), ValueError, "positions"),
    (dict(slot_mapping=torch.arange(4)), ValueError, "slot_mapping"),
    (dict(slot_mapping=torch.zeros(3)), TypeError, "integer index"),
    (dict(inv_freq=torch.ones(9)), ValueError, "inv_freq"),
    (dict(inv_freq=torch.ones(0)), ValueError, "inv_freq"),
    (dict(q_weight=W), ValueError, "together"),
    (dict(q_weight=W[:8], k_weight=W), ValueError, "shape"),
    (dict(q_weight=W.float(), k_weight=W), ValueError, "dtype"),
    (dict(out=torch.zeros(3, 4, 8, dtype=torch.bfloat16)), ValueError, "out must be"),
    (dict(), RuntimeError, "HIP devices")])
def test_qk_norm_rope_write(change, error, needle):
    with pytest.raises(error, match=needle):
        pre_attention.qk_norm_rope_write(**rope_args(**change))


@pytest.mark.parametrize("args,needle", [
    (dict(rotary_dim=7), "even"), (dict(rotary_dim=0), "even"), (dict(rotary_dim=8, base=0), "base"),
    (dict(rotary_dim=8, factor=0.5), "factor"), (dict(rotary_dim=8, factor=math.nan), "factor"),
    (dict(rotary_dim=8, scaling="other"), "unknown"),
    (dict(rotary_dim=2, scaling="ntk", factor=2.0), "at least 4"),
    (dict(rotary_dim=8, scaling="yarn", factor=2.0), "original_max_position"),
    (dict(rotary_dim=8, scaling="yarn", original_max_position=10, beta_fast=1.0), "beta_fast")])
def test_rotary_frequencies_refusals(args, needle):
    with pytest.raises(ValueError, match=needle):
        pre_attention.rotary_frequencies(**args)


def test_rotary_frequencies():
    plain, one = pre_attention.rotary_frequencies(64, 1e4)
    want = 1e4 ** (-torch.arange(32, dtype=torch.float64) / 32)
    assert torch.equal(plain, want.float()) and one == 1.0 and plain.dtype == torch.float32
    linear, one = pre_attention.rotary_frequencies(64, 1e4, scaling="linear", factor=4.0)
    assert torch.equal(linear, (want / 4).float()) and one == 1.0
    ntk, one = pre_attention.rotary_frequencies(64, 1e4, scaling="ntk", factor=4.0)
    # The fastest pair is as it was and the slowest slowed down by the factor.
    assert ntk[0] == 1.0 and one == 1.0
    assert abs(float(ntk[-1] / linear[-1]) - 1) < 1e-6
    yarn, m = pre_attention.rotary_frequencies(64, 1e4, scaling="yarn", factor=4.0,
                                               original_max_position=4096)
    turns = 4096 * want / (2 * math.pi)
    # Clear of the two ends by an index, as these are rounded outwards.
    fast, slow = int((turns > 32).sum()) - 1, int((turns >= 1).sum()) + 1
    assert torch.equal(yarn[:fast], plain[:fast]) and torch.equal(yarn[slow:], linear[slow:])
    between = yarn[fast:slow]
    assert (between <= plain[fast:slow]).all() and (between >= linear[fast:slow]).all()
    assert m == 0.1 * math.log(4.0) + 1.0
    assert pre_attention.rotary_frequencies(64, 1e4, scaling="yarn",
                                            original_max_position=4096)[1] == 1.0


def attention_args(**change):
    a = dict(q=torch.zeros(3, 4, 16, dtype=torch.bfloat16),
             k_cache=torch.zeros(4, BS, 2, 16, dtype=torch.bfloat16),
             v_cache=torch.zeros(4, BS, 2, 16, dtype=torch.bfloat16), block_size=BS)
    a.update(change)
    return a


SHARED = [
    (dict(q=torch.zeros(3, 64)), ValueError, "q must have shape"),
    (dict(k_cache=torch.zeros(4, BS, 16)), ValueError, "k_cache and v_cache must have shape"),
    (dict(v_cache=torch.zeros(3, BS, 2, 16)), ValueError, "same shape"),
    (dict(q=torch.zeros(3, 4, 32, dtype=torch.bfloat16)), ValueError, "same head_dim"),
    (dict(q=torch.zeros(3, 3, 16, dtype=torch.bfloat16)), ValueError, "divisible"),
    (dict(block_size=8), ValueError, "block_size"),
    (dict(q=torch.zeros(3, 4, 16)), TypeError, "one dtype"),
    (dict(q=torch.zeros(3, 4, 16, dtype=torch.float64)), TypeError, "unsupported dtype"),
    (dict(softcap=-1.0), ValueError, "softcap"),
    (dict(softcap=math.nan), ValueError, "softcap"),
    (dict(softcap=math.inf), ValueError, "softcap"),
    (dict(softcap=1e-31), ValueError, "softcap"),
    (dict(alibi_slopes=torch.ones(3)), ValueError, "alibi_slopes"),
    (dict(alibi_slopes=torch.ones(4, dtype=torch.bfloat16)), ValueError, "alibi_slopes"),
    (dict(), RuntimeError, "HIP devices"),
] + [(dict(q=torch.zeros(3, 4, d, dtype=t), k_cache=torch.zeros(4, BS, 2, d, dtype=t),
           v_cache=torch.zeros(4, BS, 2, d, dtype=t)), ValueError, "head_dim in multiples")
     for d, t in ((12, torch.bfloat16), (136, torch.float16), (6, torch.float32),
                  (256, torch.float32))]


@pytest.mark.parametrize("change,error,needle", SHARED)
def test_scored_attention(change, error, needle):
    a = attention_args(**change)
    bt, three = torch.zeros(3, 2, dtype=torch.long), torch.tensor([1, 2, 3])
    with pytest.raises(error, match=needle):
        scored_attention.paged_attention_decode_scored(**a, block_tables=bt, seq_lens=three)
    with pytest.raises(error, match=needle):
        scored_attention.paged_attention_prefill_scored(
            **a, block_tables=bt, query_start_loc=torch.arange(4), context_lens=three)
    with pytest.raises(error, match=needle):
        scored_attention.paged_attention_decode_shared_prefix(
            **a, prefix_table=bt[0], prefix_len=5, block_tables=bt, seq_lens=three)


def test_prefill_metadata():
    def check(qsl=(0, 2, 5), ctx=(4, 40), bt=((0, -1, -1), (1, 2, 3)), ahead=None, total=5):
        scored_attention._validate_prefill(
            torch.tensor(bt), torch.tensor(qsl), torch.tensor(ctx),
            None if ahead is None else torch.tensor(ahead), BS, 4, total)

    check()
    check(ahead=(4, 0))
    check(qsl=(0, 0, 5), ctx=(0, 40))
    for change, needle in [
            (dict(qsl=(1, 2, 5)), "start at 0"), (dict(qsl=(0, 6, 5)), "not decrease"),
            (dict(total=6), "end at the packed"), (dict(ctx=(1, 40)), "cover each"),
            (dict(ctx=(4, 49)), "insufficient blocks"),
            (dict(bt=((0, -1, -1), (1, 4, 3))), "invalid physical block"),
            (dict(bt=((-1, 0, 0), (1, 2, 3))), "invalid physical block"),
            (dict(ahead=(5, 0)), "prefix_lens"), (dict(ahead=(0, -1)), "prefix_lens")]:
        with pytest.raises(ValueError, match=needle):
            check(**change)


def sample_args(**change):
    a = dict(logits=torch.zeros(3, 50), uniforms=torch.zeros(3))
    a.update(change)
    return a


@pytest.mark.parametrize("change,error,needle", [
    (dict(logits=torch.zeros(3, 4, 50)), ValueError, "logits must have shape"),
    (dict(logits=torch.zeros(3, 0)), ValueError, "logits must have shape"),
    (dict(logits=torch.zeros(3, 50, dtype=torch.float64)), TypeError, "not supported"),
    (dict(logits=torch.zeros(3, 1).expand(3, (1 << 23) + 1)), ValueError, "2\\^23"),
    (dict(logits=torch.zeros(50, 3).T), ValueError, "unit-stride"),
    (dict(logits=torch.zeros(50).expand(3, 50)), ValueError, "overlap"),
    (dict(uniforms=torch.zeros(3, 1)), ValueError, "uniforms"),
    (dict(uniforms=torch.zeros(3).half()), ValueError, "uniforms"),
    (dict(uniforms=torch.zeros(4)), ValueError, "one number per"),
    (dict(rows=torch.zeros(2, dtype=torch.long)), ValueError, "rows"),
    (dict(rows=torch.zeros(3, dtype=torch.int32)), ValueError, "rows"),
    (dict(temperature=torch.ones(2)), ValueError, "temperature"),
    (dict(temperature=torch.ones(3).double()), ValueError, "temperature"),
    (dict(top_k=torch.ones(3)), ValueError, "top_k"),
    (dict(top_p=torch.ones(3, 1)), ValueError, "top_p"),
    (dict(min_p=torch.ones(3, dtype=torch.long)), ValueError, "min_p"),
    (dict(), RuntimeError, "HIP devices")])
def test_sample_tokens(change, error, needle):
    with pytest.raises(error, match=needle):
        sampling.sample_tokens(**sample_args(**change))


def test_random_sample():
    batch = model_runner.ModelBatch(
        request_ids=["a", "b"], input_token_ids=torch.zeros(3, dtype=torch.long),
        positions=torch.zeros(3, dtype=torch.long), query_start_loc=torch.tensor([0, 2, 3]),
        request_phases=[], context_lens=torch.ones(2), block_tables=torch.zeros(2, 1),
        slot_mapping=torch.zeros(3))
    u = torch.zeros(2)
    for logits, numbers, needle in [(torch.zeros(3), u, "packed_logits must have"),
                                    (torch.zeros(4, 9), u, "must match ModelBatch"),
                                    (torch.zeros(3, 9), torch.zeros(3), "one number per")]:
        with pytest.raises(ValueError, match=needle):
            model_runner.random_sample(logits, batch, numbers)


P = 1 << 20  # an address that nothing reads


def rope_abi(lib, **change):
    a = dict(qkv=P, st=128, qw=None, kw=None, eps=1e-6, pos=P, freq=P, rot=16, inter=0, factor=1.0,
             slots=P, index=1, out=P, ost=64, k=P, v=P, num_slots=32, tokens=3, hq=4, hkv=2, d=16,
             dtype=2, stream=None)
    a.update(change)
    return lib.mlr_qk_norm_rope_write(*a.values())


@pytest.mark.parametrize("change,needle", [
    (dict(tokens=-1), b"num_tokens"), (dict(hq=0), b"head counts"), (dict(d=15), b"even"),
    (dict(d=2048, st=1 << 20, ost=1 << 20), b"1024"), (dict(rot=18), b"rotary_dim"),
    (dict(rot=7), b"rotary_dim"), (dict(st=100), b"row stride"), (dict(ost=10), b"row stride"),
    (dict(index=7), b"index dtype"), (dict(qw=P), b"together"), (dict(pos=None), b"null"),
    (dict(hq=1 << 40), b"too wide"),
    # Odd rows of a large head: more lanes than a wave.
    (dict(d=512, rot=512, st=512 * 8 + 1, ost=2048), b"aligned")])
def test_rope_abi(change, needle):
    lib = _lib.load()
    assert rope_abi(lib, **change) == 1 and needle in lib.mlr_last_error()
    assert rope_abi(lib, dtype=3) == 2 or b"unsupported dtype" in lib.mlr_last_error()


def decode_abi(lib, **change):
    a = dict(q=P, qb=64, qh=16, k=P, v=P, nb=4, bs=BS, hkv=2, d=16, bt=P, bst=2, width=2, lens=P,
             batch=3, hq=4, scale=0.25, cap=0.0, slopes=None, dtype=2, ws=None, nbytes=0, out=P,
             ob=64, oh=16, stream=None)
    a.update(change)
    return lib.mlr_paged_decode_scored(*a.values())


@pytest.mark.parametrize("change,needle", [
    (dict(dtype=3), b"dtype"), (dict(batch=-1), b"sequences"), (dict(hq=3), b"multiple"),
    (dict(hkv=0), b"multiple"), (dict(d=20), b"head_dim"), (dict(d=136), b"head_dim"),
    (dict(nb=0), b"blocks"), (dict(bs=0), b"blocks"), (dict(width=1 << 31), b"2^31 positions"),
    (dict(cap=-1.0), b"softcap"), (dict(cap=math.nan), b"softcap"), (dict(cap=1e31), b"softcap"),
    (dict(scale=math.inf), b"scale"), (dict(qb=60), b"16 bytes"), (dict(q=P + 2), b"16 bytes"),
    (dict(k=P + 8), b"aligned"), (dict(lens=None), b"null"), (dict(bt=None), b"null"),
    (dict(width=100), b"workspace"), (dict(width=100, ws=P, nbytes=64), b"workspace")])
def test_decode_abi(change, needle):
    lib = _lib.load()
    assert decode_abi(lib, **change) == 1 and needle in lib.mlr_last_error()


def test_prefill_and_shared_abi():
    lib = _lib.load()

    def prefill(**change):
        a = dict(q=P, qb=64, qh=16, k=P, v=P, nb=4, bs=BS, hkv=2, d=16, bt=P, bst=2, width=2, qsl=P,
                 lens=P, ahead=None, seqs=3, total=9, longest=5, hq=4, scale=0.25, cap=0.0,
                 slopes=None, dtype=2, ws=None, nbytes=0, out=P, ob=64, oh=16, stream=None)
        a.update(change)
        return lib.mlr_paged_prefill_scored(*a.values())

    for change, needle in [(dict(total=-1), b"token counts"), (dict(qsl=None), b"null"),
                           (dict(longest=1 << 40, total=1 << 40), b"too many query rows"),
                           (dict(width=1000), b"workspace")]:
        assert prefill(**change) == 1 and needle in lib.mlr_last_error()
    assert prefill(total=0) == 0 and prefill(seqs=0) == 0 and prefill(longest=0) == 0

    def shared(**change):
        a = dict(q=P, qb=64, qh=16, k=P, v=P, nb=4, bs=BS, hkv=2, d=16, pt=P, pb=3, plen=40, bt=P,
                 bst=2, width=2, lens=P, batch=3, hq=4, scale=0.25, cap=0.0, slopes=None, dtype=2,
                 ws=None, nbytes=0, out=P, ob=64, oh=16, stream=None)
        a.update(change)
        return lib.mlr_paged_decode_shared_prefix(*a.values())

    for change, needle in [(dict(plen=-1), b"cover"), (dict(plen=49), b"cover"),
                           (dict(pb=1 << 40), b"cover"), (dict(pt=None), b"null"),
                           (dict(), b"workspace")]:
        assert shared(**change) == 1 and needle in lib.mlr_last_error()
    assert shared(batch=0) == 0


def test_sample_abi():
    lib = _lib.load()

    def sample(**change):
        a = dict(logits=P, st=100, total=3, dtype=0, rows=None, u=P, f64=0, t=None, tv=1.0, k=None,
                 kd=1, kv=0, p=None, pv=1.0, m=None, mv=0.0, tokens=P, lp=None, count=3, vocab=100,
                 ws=None, nbytes=0, stream=None)
        a.update(change)
        return lib.mlr_sample_tokens(*a.values())

    for change, needle in [
            (dict(count=-1), b"num_rows"), (dict(vocab=0), b"vocab"),
            (dict(vocab=(1 << 23) + 1, st=1 << 24), b"vocab"), (dict(total=2), b"fewer"),
            (dict(st=99), b"stride"), (dict(k=P, kd=5), b"index dtype"), (dict(dtype=3), b"dtype"),
            (dict(logits=None), b"null"), (dict(vocab=50000, st=50000), b"workspace"),
            (dict(vocab=50000, st=50000, ws=P + 4, nbytes=1 << 30), b"workspace")]:
        assert sample(**change) == 1 and needle in lib.mlr_last_error()
    assert sample(count=0) == 0
    assert lib.mlr_sample_tokens_workspace_size(0, 50000) == 0
    assert lib.mlr_sample_tokens_workspace_size(256, 50000) == 0
    assert lib.mlr_sample_tokens_workspace_size(4, 50000) > 0
