"""Operators of a served step whose attention is not the plain one, as cases to time.

Kinds of a case, each one pass through a public entry point:

- rope:   qk_norm_rope_write: RMSNorm of each q and k head, rotary positions
          (half or interleaved, whole head or part of it) and the append of k
          and v to the paged cache.
- prefill: paged_attention_prefill_scored: packed prompt chunks whose scores
          are capped by a tanh or biased by distance, with a prefix seen whole.
- decode: paged_attention_decode_scored: the same scores for single tokens.
- shared: paged_attention_decode_shared_prefix: a decode batch over one long
          prefix that all its requests share, and a suffix of each one's own.
- sample: sample_tokens: temperature, top-k, top-p and min-p with one given
          random number a row.

Where ``own`` is false the operators are computed in plain torch operations,
in 32 bits (angles and everything about sampling in 64), rounded once at the
end. Sizes are those of this repository's workloads and benchmarks
(Qwen2.5-0.5B: 14 query / 2 KV heads of 64, vocabulary 151936; Qwen2.5-7B:
28 / 4 heads of 128; the decode benchmark's 32 / 8 heads of 128) and generic
ones between them.
"""

import math
import os
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
BLOCK = 16
DEVICE = "cuda"


def listed() -> list:
    return [
        # One request's decode step: latency alone.
        dict(name="rope_bf16_1", kind="rope", dtype="bf16", tokens=1, hq=14, hkv=2, d=64, rot=64,
             interleaved=False, norm=True, far=32768),
        # A chunk of a prefill step at the larger model's heads.
        dict(name="rope_bf16_4096", kind="rope", dtype="bf16", tokens=4096, hq=28, hkv=4, d=128,
             rot=128, interleaved=False, norm=True, far=32768),
        # FP32, interleaved pairs over part of an odd head size, far positions
        # of a stretched context, a ragged token count.
        dict(name="rope_fp32_777_part", kind="rope", dtype="fp32", tokens=777, hq=8, hkv=2, d=96,
             rot=64, interleaved=True, norm=True, far=1000000),
        # Chunked prefill of several requests at once, capped scores.
        dict(name="prefill_cap_bf16_8x512", kind="prefill", dtype="bf16", seqs=8, q_lo=512,
             q_hi=512, past_lo=0, past_hi=3584, cap=50.0, alibi=False, ahead=0, hq=14, hkv=2,
             d=64),
        # Ragged prompts with a bias by distance, their first tokens seen whole.
        dict(name="prefill_bias_fp16_3", kind="prefill", dtype="fp16", seqs=3, q_lo=100, q_hi=1500,
             past_lo=0, past_hi=700, cap=0.0, alibi=True, ahead=400, hq=28, hkv=4, d=128),
        # An ordinary serving batch's decode with capped scores.
        dict(name="decode_cap_bf16_b64", kind="decode", dtype="bf16", batch=64, ctx_lo=128,
             ctx_hi=4096, cap=30.0, alibi=False, hq=14, hkv=2, d=64),
        # A few requests in FP32 over one short prefix that ends inside a block.
        dict(name="shared_fp32_b5", kind="shared", dtype="fp32", batch=5, prefix=300, own_lo=1,
             own_hi=90, cap=0.0, alibi=False, hq=14, hkv=2, d=64),
        # A serving batch under one long system prompt.
        dict(name="shared_bf16_b64_8k", kind="shared", dtype="bf16", batch=64, prefix=8192,
             own_lo=1, own_hi=1024, cap=0.0, alibi=False, hq=14, hkv=2, d=64),
        # Questions to one long document at the larger heads.
        dict(name="shared_fp16_b32_24k", kind="shared", dtype="fp16", batch=32, prefix=24000,
             own_lo=20, own_hi=600, cap=0.0, alibi=False, hq=28, hkv=4, d=128),
        # One request's next token from a 16-bit head.
        dict(name="sample_bf16_1", kind="sample", dtype="bf16", rows=1, vocab=151936, topk=True,
             topp=True, minp=False),
        # FP32 logits of an ordinary batch, every filter.
        dict(name="sample_fp32_48", kind="sample", dtype="fp32", rows=48, vocab=151936, topk=True,
             topp=True, minp=True),
        # A large batch, nucleus alone: whole rows carry weight.
        dict(name="sample_bf16_256_topp", kind="sample", dtype="bf16", rows=256, vocab=151936,
             topk=False, topp=True, minp=False),
    ]


def _log(rng, lo, hi) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


# (query heads, KV heads, head_dim): what the tests and benchmarks run most,
# and others that a configuration may give.
HEADS = [(14, 2, 64), (14, 2, 64), (28, 4, 128), (32, 8, 128), (12, 12, 64), (16, 1, 128),
         (4, 2, 16), (8, 2, 96), (6, 3, 32), (10, 2, 80)]


def draw(rng) -> dict:
    kind = rng.choice(["rope", "prefill", "decode", "shared", "sample"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    hq, hkv, d = rng.choice(HEADS)
    heads = dict(hq=hq, hkv=hkv, d=d)
    if kind == "rope":
        return dict(kind=kind, dtype=dtype, tokens=_log(rng, 1, 4096 if dtype != "fp32" else 2048),
                    rot=max(2, rng.choice([d, d, d // 2, d // 4 * 2])),
                    interleaved=rng.random() < 0.5, norm=rng.random() < 0.75,
                    far=_log(rng, 64, 1000000), **heads)
    if kind == "sample":
        rows = _log(rng, 1, 256)
        return dict(kind=kind, dtype=dtype, rows=rows,
                    vocab=_log(rng, 100, min(151936, 151936 * 256 // rows)),
                    topk=rng.random() < 0.5, topp=rng.random() < 0.6, minp=rng.random() < 0.4)
    cap = rng.choice([0.0, 20.0, 50.0])
    alibi = rng.random() < 0.5
    if kind == "prefill":
        seqs = _log(rng, 1, 12)
        rows = (2048 if dtype != "fp32" else 512) * 896 // max(896, hq * d)
        q_hi = _log(rng, 2, max(32, rows // seqs))
        return dict(kind=kind, dtype=dtype, seqs=seqs,
                    q_lo=max(1, int(q_hi * rng.uniform(0.1, 1))), q_hi=q_hi, past_lo=0,
                    past_hi=_log(rng, 16, 2048), cap=cap, alibi=alibi,
                    ahead=rng.choice([0, _log(rng, 1, 1000)]), **heads)
    row = 2 * hkv * d * SIZE[dtype]  # bytes of one position's K and V
    if kind == "decode":
        batch = _log(rng, 1, 96)
        hi = _log(rng, 16, max(64, min(16384, 70000000 // (row * batch))))
        return dict(kind=kind, dtype=dtype, batch=batch,
                    ctx_lo=max(1, int(hi * rng.uniform(0.03, 1.0))), ctx_hi=hi, cap=cap,
                    alibi=alibi, **heads)
    batch = _log(rng, 1, 64)
    own_hi = _log(rng, 1, max(16, min(1024, 35000000 // (row * batch))))
    return dict(kind=kind, dtype=dtype, batch=batch,
                prefix=_log(rng, 16, min(16384 if dtype != "fp32" else 4096, 35000000 // row)),
                own_lo=max(1, int(own_hi * rng.uniform(0.02, 1.0))), own_hi=own_hi, cap=cap,
                alibi=alibi, **heads)


# ---------------------------------------------------------------------------
# Sizes that follow from a case alone
# ---------------------------------------------------------------------------
def _lengths(n, lo, hi, salt) -> list:
    """n lengths over [lo, hi], the longest among them."""
    rng = random.Random(7919 * n + 31 * lo + hi + salt)
    lens = [rng.randint(lo, hi) for _ in range(n)]
    lens[rng.randrange(n)] = hi
    return lens


def _chunks(case) -> list:
    """[(past, queries)] of a prefill case's sequences."""
    return list(zip(_lengths(case["seqs"], case["past_lo"], case["past_hi"], 3),
                    _lengths(case["seqs"], case["q_lo"], case["q_hi"], 2)))


def work(case) -> dict:
    kind, size = case["kind"], SIZE[case["dtype"]]
    if kind == "sample":
        # Each logit: its distance, weight and place in a sum.
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + 32 * case["rows"], "flops": 10 * n}
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if kind == "rope":
        # Rows read and written once; a position and a slot a token.
        n = case["tokens"] * (hq + 2 * hkv) * d
        return {"bytes": 2 * n * size + 16 * case["tokens"] + 2 * d * size + 2 * case["rot"],
                "flops": 10 * n}
    if kind == "prefill":
        rows = keys = pairs = 0
        for past, n in _chunks(case):
            ctx, ahead = past + n, min(case["ahead"], past + n)
            rows, keys = rows + n, keys + ctx
            pairs += sum(max(past + i + 1, ahead) for i in range(n))
    elif kind == "decode":
        lens = _lengths(case["batch"], case["ctx_lo"], case["ctx_hi"], 1)
        rows, keys, pairs = len(lens), sum(lens), sum(lens)
    else:
        lens = _lengths(case["batch"], case["own_lo"], case["own_hi"], 1)
        rows, keys = len(lens), case["prefix"] + sum(lens)
        pairs = sum(lens) + len(lens) * case["prefix"]
    return {"bytes": (2 * rows * hq + 2 * keys * hkv) * d * size + 8 * keys // BLOCK,
            "flops": 4 * d * hq * pairs}


# ---------------------------------------------------------------------------
# prepare
# ---------------------------------------------------------------------------
def _long(values):
    return torch.tensor(values, dtype=torch.long, device=DEVICE)


def _tables(lens, seed):
    """(block tables as lists from a shuffled pool, blocks in the pool)."""
    need = [-(-n // BLOCK) for n in lens]
    total = sum(need) + 1 + sum(need) // 8
    perm = list(range(total))
    random.Random(seed).shuffle(perm)
    tables, at = [], 0
    for n in need:
        tables.append(perm[at:at + n])
        at += n
    return tables, total


def _padded(tables):
    width = max(len(t) for t in tables)
    return _long([t + [-1] * (width - len(t)) for t in tables])


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed))
    dtype, kind = DTYPES[case["dtype"]], case["kind"]

    def rand(*shape, scale=1.0):
        return (torch.randn(shape, generator=gen, device=DEVICE) * scale).to(dtype)

    s = {"case": case}
    if kind == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # Gumbel-shaped logits: rows from a few likely tokens to broad ones.
        u = torch.rand(rows, vocab, generator=gen, device=DEVICE).clamp_(1e-7, 1 - 1e-7)
        spread = 0.6 + 1.4 * torch.rand(rows, 1, generator=gen, device=DEVICE)
        s["logits"] = (-(-u.log()).log() * spread).to(dtype)
        s["uniforms"] = torch.rand(rows, generator=gen, device=DEVICE)
        pick = torch.rand(4, rows, generator=gen, device=DEVICE)
        # One row in eight is decoded greedily.
        s["temperature"] = torch.where(pick[0] < 0.125, 0.0, 0.5 + 0.8 * pick[0])
        choices = _long([1, 5, 20, 50, 200, 1000])
        s["top_k"] = choices[(pick[1] * 6).long().clamp_(max=5)] if case["topk"] else None
        s["top_p"] = 0.7 + 0.29 * pick[2] if case["topp"] else None
        s["min_p"] = 0.1 * pick[3] if case["minp"] else None
        return s
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if kind == "rope":
        tokens, half = case["tokens"], case["rot"] // 2
        blocks = -(-tokens // BLOCK) + 1
        s["k_cache"], s["v_cache"] = rand(blocks, BLOCK, hkv, d), rand(blocks, BLOCK, hkv, d)
        s["qkv"] = rand(tokens, (hq + 2 * hkv) * d)
        s["q_weight"] = 1 + rand(d, scale=0.1) if case["norm"] else None
        s["k_weight"] = 1 + rand(d, scale=0.1) if case["norm"] else None
        # Low frequencies slowed down four times, as for a stretched context.
        freq = 1e6 ** (-torch.arange(half, dtype=torch.float64, device=DEVICE) / half)
        s["inv_freq"] = torch.where(freq < 1e-3, freq / 4, freq).float()
        start = torch.randint(0, case["far"], (), generator=gen, device=DEVICE)
        s["positions"] = (start + torch.arange(tokens, device=DEVICE)) % case["far"]
        s["slots"] = torch.randperm(blocks * BLOCK, generator=gen, device=DEVICE)[:tokens]
        s["factor"] = 1.1
        return s
    s["scale"] = d ** -0.5
    s["cap"] = case["cap"]
    s["slopes"] = (2.0 ** (-8.0 * torch.arange(1, hq + 1, device=DEVICE) / hq)
                   if case["alibi"] else None)
    if kind == "prefill":
        chunks = _chunks(case)
        lens, qs = [p + n for p, n in chunks], [n for _, n in chunks]
        rows = sum(qs)
        s["qsl"] = _long([sum(qs[:i]) for i in range(len(qs) + 1)])
        s["max_q"] = max(qs)
        s["ahead"] = _long([min(case["ahead"], n) for n in lens]) if case["ahead"] else None
    elif kind == "decode":
        lens = _lengths(case["batch"], case["ctx_lo"], case["ctx_hi"], 1)
        rows = len(lens)
    else:
        suffix = _lengths(case["batch"], case["own_lo"], case["own_hi"], 1)
        lens, rows, prefix = [case["prefix"] + n for n in suffix], len(suffix), case["prefix"]
    if kind == "shared":
        # Whole blocks of the prefix are the same in every table; from the
        # block in which it ends on, each request has its own.
        whole = prefix // BLOCK
        tables, blocks = _tables([prefix] + [n - whole * BLOCK for n in lens], seed)
        s["prefix_table"] = _long(tables[0])
        tables = [tables[0][:whole] + t for t in tables[1:]]
        s["prefix"] = prefix
    else:
        tables, blocks = _tables(lens, seed)
    s["k"], s["v"] = rand(blocks, BLOCK, hkv, d), rand(blocks, BLOCK, hkv, d)
    s["q"] = rand(rows, hq, d)
    s["bt"], s["ctx"], s["max_ctx"] = _padded(tables), _long(lens), max(lens)
    return s


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------
def _plain_rope(s):
    case = s["case"]
    hq, hkv, d, rot = case["hq"], case["hkv"], case["d"], case["rot"]
    tokens, dtype = s["qkv"].shape[0], s["qkv"].dtype
    q, k, v = s["qkv"].view(tokens, hq + 2 * hkv, d).split([hq, hkv, hkv], dim=1)
    angle = s["positions"].double()[:, None] * s["inv_freq"].double()[None, :]
    cos = (angle.cos() * s["factor"]).float()[:, None, :]
    sin = (angle.sin() * s["factor"]).float()[:, None, :]

    def head(x, weight):
        x = x.float()
        if weight is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight.float()
        part, rest = x[..., :rot], x[..., rot:]
        if case["interleaved"]:
            lo, hi = part[..., 0::2], part[..., 1::2]
            part = torch.stack([lo * cos - hi * sin, hi * cos + lo * sin], dim=-1).flatten(-2)
        else:
            lo, hi = part[..., :rot // 2], part[..., rot // 2:]
            part = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], dim=-1)
        return torch.cat([part, rest], dim=-1).to(dtype)

    s["k_cache"].view(-1, hkv, d).index_copy_(0, s["slots"], head(k, s["k_weight"]))
    s["v_cache"].view(-1, hkv, d).index_copy_(0, s["slots"], v)
    return head(q, s["q_weight"]), s["k_cache"], s["v_cache"]


def _keys(cache, tables, count):
    """The first `count` rows of each table's blocks: [S, Hkv, count, D] in 32 bits."""
    hkv, d = cache.shape[2:]
    rows = cache[tables.clamp(min=0)].view(tables.shape[0], -1, hkv, d)[:, :count]
    return rows.float().transpose(1, 2).contiguous()


def _scores(s, q, k, distance):
    """Scores of q [S, Hq, L, D] on k [S, Hkv, N, D]: [S, Hq, L, N]; distance
    broadcasts to [S, L, N]."""
    seqs, hq, length, d = q.shape
    hkv = k.shape[1]
    q = q.reshape(seqs, hkv, hq // hkv * length, d)
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()).view(seqs, hq, length, -1) * s["scale"]
    if s["cap"] > 0:
        x = s["cap"] * torch.tanh(x / s["cap"])
    if s["slopes"] is not None:
        x = x - s["slopes"][None, :, None, None] * distance[:, None].float()
    return x


def _values(p, v):
    """p [S, Hq, L, N] times v [S, Hkv, N, D]: [S, Hq, L, D]."""
    seqs, hq, length, n = p.shape
    hkv = v.shape[1]
    return torch.matmul(p.reshape(seqs, hkv, hq // hkv * length, n), v).view(seqs, hq, length, -1)


def _softmax(x, visible):
    x = x.masked_fill(~visible, float("-inf"))
    p = (x - x.amax(-1, keepdim=True)).exp()
    return p / p.sum(-1, keepdim=True)


def _plain_prefill(s):
    q, ctx, qsl = s["q"], s["ctx"], s["qsl"]
    lens = qsl[1:] - qsl[:-1]
    row = torch.arange(s["max_q"], device=q.device)
    padded = q[(qsl[:-1, None] + row).clamp(max=q.shape[0] - 1)].float().transpose(1, 2)
    k, v = _keys(s["k"], s["bt"], s["max_ctx"]), _keys(s["v"], s["bt"], s["max_ctx"])
    key = torch.arange(s["max_ctx"], device=q.device)[None, None, :]
    # Padding rows stand at the last position, so that they see a key too.
    pos = torch.minimum((ctx - lens)[:, None] + row, ctx[:, None] - 1)[:, :, None]
    limit = pos + 1
    if s["ahead"] is not None:
        limit = torch.maximum(limit, s["ahead"][:, None, None])
    p = _softmax(_scores(s, padded, k, (pos - key).abs()), (key < limit)[:, None])
    out = _values(p, v).transpose(1, 2)  # [S, L, Hq, D]
    token = torch.arange(q.shape[0], device=q.device)
    owner = torch.searchsorted(qsl[1:].contiguous(), token, right=True)
    return out[owner, token - qsl[owner]].to(q.dtype)


def _plain_decode(s):
    q, ctx = s["q"], s["ctx"]
    k, v = _keys(s["k"], s["bt"], s["max_ctx"]), _keys(s["v"], s["bt"], s["max_ctx"])
    key = torch.arange(s["max_ctx"], device=q.device)[None, None, :]
    distance = ctx[:, None, None] - 1 - key
    p = _softmax(_scores(s, q.float()[:, :, None], k, distance), (distance >= 0)[:, None])
    return _values(p, v)[:, :, 0].to(q.dtype)


def _plain_shared(s):
    q, ctx, prefix = s["q"], s["ctx"], s["prefix"]
    first = prefix // BLOCK
    skip = prefix - first * BLOCK
    count = s["max_ctx"] - first * BLOCK
    kp, vp = _keys(s["k"], s["prefix_table"][None], prefix), _keys(s["v"], s["prefix_table"][None],
                                                                  prefix)
    ks, vs = _keys(s["k"], s["bt"][:, first:], count), _keys(s["v"], s["bt"][:, first:], count)
    key = torch.arange(prefix, device=q.device)[None, None, :]
    own_key = (first * BLOCK + torch.arange(count, device=q.device))[None, None, :]
    last = ctx[:, None, None] - 1
    # All requests' rows at once over the prefix: [1, Hq, B, D].
    over = _scores(s, q.float().transpose(0, 1)[None], kp, (ctx[None, :, None] - 1 - key))
    rest = _scores(s, q.float()[:, :, None], ks, last - own_key)[:, :, 0]
    x = torch.cat([over[0].transpose(0, 1), rest], dim=-1)  # [B, Hq, prefix + count]
    visible = (own_key <= last) & (own_key >= first * BLOCK + skip)
    visible = torch.cat([torch.ones_like(visible[:, :, :1]).expand(-1, -1, prefix), visible], -1)
    p = _softmax(x, visible)
    out = _values(p[None, :, :, :prefix].transpose(1, 2), vp)[0].transpose(0, 1)
    out = out + _values(p[:, :, None, prefix:], vs)[:, :, 0]
    return out.to(q.dtype)


def _plain_sample(s):
    x = s["logits"].double()
    rows, vocab = x.shape
    x = x.masked_fill(x.isnan(), float("-inf"))
    x, order = torch.sort(x, dim=-1, descending=True, stable=True)
    rank = torch.arange(vocab, device=x.device)[None]
    greedy = s["temperature"][:, None] == 0
    t = torch.where(greedy, 1.0, s["temperature"][:, None].double())
    w = torch.where(x == x[:, :1], 1.0, ((x - x[:, :1]) / t).exp())
    w = w.masked_fill(x == float("-inf"), 0.0)
    keep = ~greedy | (rank == 0)
    if s["top_k"] is not None:
        keep = keep & ((rank < s["top_k"][:, None]) | (s["top_k"][:, None] <= 0))
    w = w * keep
    if s["top_p"] is not None:
        before = w.cumsum(-1) - w
        p = s["top_p"][:, None].double()
        w = w * ((before < p * w.sum(-1, keepdim=True)) | (rank == 0) | (p >= 1))
    if s["min_p"] is not None:
        w = w * ((w >= s["min_p"][:, None].double()) | (rank == 0))
    cdf = w.cumsum(-1)
    target = s["uniforms"][:, None].double() * cdf[:, -1:]
    at = torch.searchsorted(cdf, target, right=True)
    # A target that rounding put on the sum: the last token with weight.
    at = torch.minimum(at, torch.where(w > 0, rank, -1).amax(-1, keepdim=True))
    none = at[:, 0] < 0
    at = at.clamp(min=0)
    logprob = (w.gather(-1, at) / cdf[:, -1:]).log().float()[:, 0]
    token = order.gather(-1, at)[:, 0]
    return token.masked_fill(none, -1), logprob.masked_fill(none, float("-inf"))


# ---------------------------------------------------------------------------
# The framework's own
# ---------------------------------------------------------------------------
_own = {}


def _calls():
    if not _own:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        sys.path.insert(1, os.path.join(root, "mini-llm-runtime_amd"))
        from mini_llm_runtime_amd.kernels import pre_attention, sampling, scored_attention

        _own.update(rope=pre_attention.qk_norm_rope_write, sample=sampling.sample_tokens,
                    prefill=scored_attention.paged_attention_prefill_scored,
                    decode=scored_attention.paged_attention_decode_scored,
                    shared=scored_attention.paged_attention_decode_shared_prefix)
    return _own


def _run_own(s):
    case = s["case"]
    kind = case["kind"]
    call = _calls()[kind]
    if kind == "rope":
        q = call(s["qkv"], s["positions"], s["inv_freq"], s["k_cache"], s["v_cache"], s["slots"],
                 case["hq"], q_weight=s["q_weight"], k_weight=s["k_weight"], eps=1e-6,
                 interleaved=case["interleaved"], attention_factor=s["factor"])
        return q, s["k_cache"], s["v_cache"]
    if kind == "sample":
        # A filter that is off has its neutral value.
        return call(s["logits"], s["uniforms"], temperature=s["temperature"],
                    top_k=0 if s["top_k"] is None else s["top_k"],
                    top_p=1.0 if s["top_p"] is None else s["top_p"],
                    min_p=0.0 if s["min_p"] is None else s["min_p"], return_logprobs=True)
    # The step's metadata is checked once a step, not in every layer.
    if kind == "prefill":
        return call(s["q"], s["k"], s["v"], s["bt"], s["qsl"], s["ctx"], BLOCK,
                    softcap=s["cap"], alibi_slopes=s["slopes"], prefix_lens=s["ahead"],
                    scale=s["scale"], max_query_len=s["max_q"], validate=False)
    if kind == "decode":
        return call(s["q"], s["k"], s["v"], s["bt"], s["ctx"], BLOCK, softcap=s["cap"],
                    alibi_slopes=s["slopes"], scale=s["scale"], validate=False)
    return call(s["q"], s["k"], s["v"], s["prefix_table"], s["prefix"], s["bt"], s["ctx"], BLOCK,
                softcap=s["cap"], alibi_slopes=s["slopes"], scale=s["scale"], validate=False)


_PLAIN = {"rope": _plain_rope, "prefill": _plain_prefill, "decode": _plain_decode,
          "shared": _plain_shared, "sample": _plain_sample}


def run(s):
    if own:
        return _run_own(s)
    return _PLAIN[s["case"]["kind"]](s)


# ---------------------------------------------------------------------------
# The definitions in 64 bits, row by row
# ---------------------------------------------------------------------------
def _exact_rope(s):
    case = s["case"]
    hq, hkv, d, rot = case["hq"], case["hkv"], case["d"], case["rot"]
    x = s["qkv"].double().view(-1, hq + 2 * hkv, d)
    angle = torch.outer(s["positions"].double(), s["inv_freq"].double())
    turn = torch.polar(torch.full_like(angle, s["factor"]), angle)[:, None, :]
    out = []
    for part, weight in ((x[:, :hq], s["q_weight"]), (x[:, hq:hq + hkv], s["k_weight"])):
        n = part.clone()
        if weight is not None:
            n = n / ((n ** 2).sum(-1, keepdim=True) / d + 1e-6) ** 0.5 * weight.double()
        # Each rotated pair as one complex number times exp(i angle).
        if case["interleaved"]:
            first, second = slice(0, rot, 2), slice(1, rot, 2)
        else:
            first, second = slice(0, rot // 2), slice(rot // 2, rot)
        z = torch.complex(n[..., first], n[..., second]) * turn
        n[..., first], n[..., second] = z.real, z.imag
        out.append(n)
    k, v = s["k_cache"].double(), s["v_cache"].double()
    k.view(-1, hkv, d)[s["slots"]] = out[1]
    v.view(-1, hkv, d)[s["slots"]] = x[:, hq + hkv:]
    return out[0], k, v


def _exact_rows(s, q, k, v, pos, limit):
    """One sequence: q [n, Hq, D] at positions pos [n], keys [N, Hkv, D] below
    limit [n]."""
    hq, group = q.shape[1], q.shape[1] // k.shape[1]
    at = torch.arange(k.shape[0], device=q.device)
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    for h in range(hq):
        kh, vh = k[:, h // group].double(), v[:, h // group].double()
        x = (q[:, h].double() @ kh.T.contiguous()) * s["scale"]
        if s["cap"]:
            x = torch.tanh(x / s["cap"]) * s["cap"]
        if s["slopes"] is not None:
            x -= float(s["slopes"][h]) * (pos[:, None] - at[None]).abs().double()
        x[at[None] >= limit[:, None]] = -math.inf
        out[:, h] = torch.softmax(x, -1) @ vh
    return out


def _exact_attention(s):
    case = s["case"]
    kind, hkv, d = case["kind"], case["hkv"], case["d"]
    lens = s["ctx"].tolist()
    starts = s["qsl"].tolist() if kind == "prefill" else list(range(len(lens) + 1))
    outs = []
    for i, n in enumerate(lens):
        slot = torch.arange(n, device=DEVICE)
        block = s["bt"][i][slot // BLOCK]
        if kind == "shared":
            p = s["prefix"]
            block = torch.cat([s["prefix_table"][slot[:p] // BLOCK], block[p:]])
        k = s["k"].view(-1, hkv, d)[block * BLOCK + slot % BLOCK]
        v = s["v"].view(-1, hkv, d)[block * BLOCK + slot % BLOCK]
        q = s["q"][starts[i]:starts[i + 1]]
        pos = n - q.shape[0] + torch.arange(q.shape[0], device=DEVICE)
        limit = pos + 1
        if kind == "prefill" and s["ahead"] is not None:
            limit = limit.clamp(min=int(s["ahead"][i]))
        outs.append(_exact_rows(s, q, k, v, pos, limit))
    return torch.cat(outs)


def _exact_sample(s):
    def value(name, row, off):
        return off if s[name] is None else s[name][row].item()

    tokens, logprobs = [], []
    for r in range(s["logits"].shape[0]):
        x = s["logits"][r].double()
        t = value("temperature", r, 1.0)
        k = value("top_k", r, 0)
        p, m = value("top_p", r, 1.0), value("min_p", r, 0.0)
        order = torch.argsort(x, descending=True, stable=True)
        if t == 0:
            tokens.append(int(order[0]))
            logprobs.append(0.0)
            continue
        w = torch.softmax(x / t, -1)
        head = order[:k] if k > 0 else order
        mass = w[head].cumsum(0)
        if p < 1:
            n = int((mass < p * mass[-1]).sum()) + 1
            head = head[:n]
        head = head[(w[head] >= m * w[order[0]]) | (head == order[0])]
        mass = w[head].cumsum(0)
        at = int((mass <= s["uniforms"][r].double() * mass[-1]).sum().clamp(max=len(head) - 1))
        tokens.append(int(head[at]))
        logprobs.append(math.log(float(w[head[at]] / mass[-1])))
    return (_long(tokens), torch.tensor(logprobs, dtype=torch.float64, device=DEVICE))


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rope":
        return _exact_rope(s)
    if case["kind"] == "sample":
        return _exact_sample(s)
    return _exact_attention(s)
