"""Operators that choose which keys of a paged cache a token sees, or which keys
it holds, as cases to time.

Kinds of a case, each one pass through a public entry point:

- tree:   paged_attention_tree: several drafted tokens a request, each seeing the
          cache and its own ancestors among the drafted ones.
- move:   compact_keys: cache rows that stay (an accepted path of drafted tokens,
          or any list per KV head) move together, in place.
- weigh:  paged_attention_decode_weighted: single-token decode that adds what each
          key's attention weights come to.
- evict:  evict_keys: by these sums, the heaviest keys stay, in place.
- bounds: update_key_bounds: the elementwise minimum and maximum of each block's
          keys.
- sparse: paged_attention_decode_sparse: single-token decode over the blocks whose
          bounds promise the largest scores.

Where ``own`` is false the operators are computed in plain torch operations, in 32
bits (the blocks' scores, which decide which blocks are read, in 64), rounded
once at the end. Sizes are those of this repository's workloads and benchmarks
(Qwen2.5-0.5B: 14 query / 2 KV heads of 64; Qwen2.5-7B: 28 / 4 heads of 128; the
decode benchmark's 32 / 8 heads of 128; blocks of 16) and generic ones between
them.
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
        # A few short drafts of FP32 requests: latency alone.
        dict(name="tree_fp32_3x9", kind="tree", dtype="fp32", seqs=3, n_lo=2, n_hi=9, past_lo=1,
             past_hi=300, cap=0.0, hq=14, hkv=2, d=64),
        # A serving batch's drafted trees at the larger model's heads.
        dict(name="tree_bf16_16x48", kind="tree", dtype="bf16", seqs=16, n_lo=20, n_hi=48,
             past_lo=512, past_hi=4096, cap=0.0, hq=28, hkv=4, d=128),
        # The accepted paths of a batch's drafted trees.
        dict(name="move_bf16_b16_path", kind="move", dtype="bf16", batch=16, ctx_lo=300,
             ctx_hi=4096, drafted=32, keep_lo=1, keep_hi=7, per_head=False, hq=14, hkv=2, d=64),
        # A quarter of long contexts dropped, other keys for every KV head.
        dict(name="move_fp16_b4_8k", kind="move", dtype="fp16", batch=4, ctx_lo=8000, ctx_hi=8192,
             drafted=0, keep_lo=6000, keep_hi=6144, per_head=True, hq=32, hkv=8, d=128),
        # A few FP32 requests, odd head size, capped scores.
        dict(name="weigh_fp32_b3", kind="weigh", dtype="fp32", batch=3, ctx_lo=1, ctx_hi=600,
             cap=20.0, hq=8, hkv=2, d=96),
        # An ordinary serving batch.
        dict(name="weigh_bf16_b64", kind="weigh", dtype="bf16", batch=64, ctx_lo=128, ctx_hi=4096,
             cap=0.0, hq=14, hkv=2, d=64),
        # A batch that has grown by a block past what it may keep.
        dict(name="evict_bf16_b64_1k", kind="evict", dtype="bf16", batch=64, ctx_lo=1030,
             ctx_hi=1040, budget=1024, sinks=4, recent=256, hq=14, hkv=2, d=64),
        # Long prompts cut to a quarter after their prefill.
        dict(name="evict_fp16_b8_16k", kind="evict", dtype="fp16", batch=8, ctx_lo=12000,
             ctx_hi=16384, budget=4096, sinks=4, recent=512, hq=28, hkv=4, d=128),
        # One decode step's new keys.
        dict(name="bounds_bf16_b64_step", kind="bounds", dtype="bf16", batch=64, ctx_lo=128,
             ctx_hi=4096, new=1, hq=14, hkv=2, d=64),
        # All blocks of long prompts.
        dict(name="bounds_fp16_b4_8k", kind="bounds", dtype="fp16", batch=4, ctx_lo=7000,
             ctx_hi=8192, new=0, hq=32, hkv=8, d=128),
        # Two FP32 requests of middling length.
        dict(name="sparse_fp32_b2_2k", kind="sparse", dtype="fp32", batch=2, ctx_lo=1500,
             ctx_hi=2047, budget=40, sinks=1, recent=2, cap=0.0, hq=14, hkv=2, d=64),
        # Long contexts, an eighth of them read, at the larger model's heads.
        dict(name="sparse_bf16_b8_32k", kind="sparse", dtype="bf16", batch=8, ctx_lo=30000,
             ctx_hi=32768, budget=256, sinks=1, recent=4, cap=0.0, hq=28, hkv=4, d=128),
    ]


def _log(rng, lo, hi) -> int:
    hi = max(lo, hi)
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


# (query heads, KV heads, head_dim): what the tests and benchmarks run most,
# and others that a configuration may give.
HEADS = [(14, 2, 64), (14, 2, 64), (28, 4, 128), (32, 8, 128), (12, 12, 64), (16, 1, 128),
         (4, 2, 16), (8, 2, 96), (6, 3, 32), (10, 2, 80)]


def draw(rng) -> dict:
    kind = rng.choice(["tree", "move", "weigh", "evict", "bounds", "sparse"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    hq, hkv, d = rng.choice(HEADS)
    case = dict(kind=kind, dtype=dtype, hq=hq, hkv=hkv, d=d)
    row = 2 * hkv * d * SIZE[dtype]  # bytes of one position's K and V
    if kind == "tree":
        seqs = _log(rng, 1, 16)
        n_hi = _log(rng, 2, 64 if hq * d <= 2048 else 40)
        past_hi = _log(rng, 16, min(4096, 60000000 // (row * seqs)))
        return dict(case, seqs=seqs, n_lo=max(1, int(n_hi * rng.uniform(0.1, 1))), n_hi=n_hi,
                    past_lo=max(1, int(past_hi * rng.uniform(0.02, 1))), past_hi=past_hi,
                    cap=rng.choice([0.0, 0.0, 50.0]))
    if kind in ("move", "evict", "bounds"):
        batch = _log(rng, 1, 64)
        hi = _log(rng, 32, min(16384, 100000000 // (row * batch)))
        case.update(batch=batch, ctx_lo=max(2, int(hi * rng.uniform(0.1, 1.0))), ctx_hi=hi)
        if kind == "bounds":
            return dict(case, new=rng.choice([0, 1, _log(rng, 1, 300)]))
        if kind == "evict":
            budget = max(16, int(hi * rng.uniform(0.2, 1.05)))
            return dict(case, budget=budget, sinks=rng.choice([0, 4]),
                        recent=int(budget * rng.uniform(0.05, 0.6)))
        if rng.random() < 0.5:
            drafted = min(case["ctx_lo"], _log(rng, 2, 64))
            keep = min(drafted, _log(rng, 1, 12))
            return dict(case, drafted=drafted, keep_lo=1, keep_hi=keep, per_head=False)
        keep = max(1, int(case["ctx_lo"] * rng.uniform(0.1, 1.0)))
        return dict(case, drafted=0, keep_lo=max(1, keep * 9 // 10), keep_hi=keep,
                    per_head=rng.random() < 0.7)
    cap = rng.choice([0.0, 0.0, 30.0])
    if kind == "weigh":
        batch = _log(rng, 1, 96)
        hi = _log(rng, 16, min(16384, 70000000 // (row * batch)))
        return dict(case, batch=batch, ctx_lo=max(1, int(hi * rng.uniform(0.03, 1.0))), ctx_hi=hi,
                    cap=cap)
    batch = _log(rng, 1, 64)
    hi = _log(rng, 64, min(65536, 400000000 // (row * batch)))
    blocks = -(-hi // BLOCK)
    budget = max(4, min(512, int(blocks * rng.uniform(0.05, 0.6))))
    return dict(case, batch=batch, ctx_lo=max(1, int(hi * rng.uniform(0.3, 1.0))), ctx_hi=hi,
                budget=budget, sinks=rng.choice([0, 1]), recent=rng.choice([1, 2]), cap=cap)


# ---------------------------------------------------------------------------
# Sizes that follow from a case alone
# ---------------------------------------------------------------------------
def _lengths(n, lo, hi, salt) -> list:
    """n lengths over [lo, hi], the longest among them."""
    rng = random.Random(7919 * n + 31 * lo + hi + salt)
    lens = [rng.randint(lo, hi) for _ in range(n)]
    lens[rng.randrange(n)] = hi
    return lens


def _trees(case) -> list:
    """[(cached tokens, drafted tokens)] of a tree case's requests."""
    return list(zip(_lengths(case["seqs"], case["past_lo"], case["past_hi"], 3),
                    _lengths(case["seqs"], case["n_lo"], case["n_hi"], 2)))


def _kept_counts(case) -> list:
    return _lengths(case["batch"], case["keep_lo"], case["keep_hi"], 5)


def _starts(case, lens) -> list:
    """The first position of each request whose key is new (bounds)."""
    return [max(0, n - case["new"]) if case["new"] else 0 for n in lens]


def work(case) -> dict:
    kind, size = case["kind"], SIZE[case["dtype"]]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    row = 2 * hkv * d * size  # K and V of one position
    if kind == "tree":
        trees = _trees(case)
        rows, keys = sum(n for _, n in trees), sum(p + n for p, n in trees)
        # A drafted token sees some 6 of the drafted ones.
        pairs = sum(n * (p + min(n, 6)) for p, n in trees)
        return {"bytes": 2 * rows * hq * d * size + keys * row + 8 * keys // BLOCK + 8 * rows,
                "flops": 4 * d * hq * pairs}
    lens = _lengths(case["batch"], case["ctx_lo"], case["ctx_hi"], 1)
    batch = case["batch"]
    if kind == "move":
        kept = sum(_kept_counts(case))
        return {"bytes": 2 * kept * row + 8 * kept * (hkv if case["per_head"] else 1) +
                         16 * kept // BLOCK, "flops": 0}
    if kind == "weigh":
        keys = sum(lens)
        return {"bytes": 2 * batch * hq * d * size + keys * row + 8 * keys // BLOCK +
                         8 * keys * hkv, "flops": 4 * d * hq * keys}
    if kind == "evict":
        # Every key's sum is read, and what moves is read and written.
        kept = sum(case["budget"] - case["sinks"] for n in lens if n > case["budget"])
        return {"bytes": 4 * hkv * sum(lens) + 2 * kept * (row + 4 * hkv) +
                         8 * hkv * batch * case["budget"] + 16 * sum(lens) // BLOCK,
                "flops": hkv * sum(lens)}
    blocks = [-(-n // BLOCK) for n in lens]
    if kind == "bounds":
        keys = changed = 0
        for n, s in zip(lens, _starts(case, lens)):
            first = s // BLOCK
            keys, changed = keys + n - first * BLOCK, changed + -(-n // BLOCK) - first
        return {"bytes": keys * row // 2 + changed * (row + 8), "flops": keys * hkv * d * 2}
    chosen = [min(b, case["budget"]) for b in blocks]
    keys = sum((c - 1) * BLOCK + (n - 1) % BLOCK + 1 for c, n in zip(chosen, lens))
    return {"bytes": 2 * batch * hq * d * size + keys * row + sum(blocks) * (row + 8) +
                     8 * batch * hkv * case["budget"],
            "flops": 4 * d * hq * (keys + sum(blocks))}


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


def _ancestor_words(counts, seed):
    """Each drafted token's ancestors and itself as bits, 64 to a word: trees whose
    later nodes hang mostly from late ones."""
    rng = random.Random(seed)
    words = -(-max(counts) // 64)
    rows = []
    for n in counts:
        seen = []
        for i in range(n):
            parent = i - 1 - min(i - 1, int(rng.expovariate(0.25))) if i else -1
            seen.append((seen[parent] if parent >= 0 else 0) | 1 << i)
        rows += seen
    def signed(word):
        return word - (1 << 64) if word >> 63 else word
    return _long([[signed(r >> 64 * w & (1 << 64) - 1) for w in range(words)] for r in rows])


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed))
    dtype, kind = DTYPES[case["dtype"]], case["kind"]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]

    def rand(*shape):
        return torch.randn(shape, generator=gen, device=DEVICE).to(dtype)

    s = {"case": case, "scale": d ** -0.5}
    if kind == "tree":
        trees = _trees(case)
        lens, counts = [p + n for p, n in trees], [n for _, n in trees]
        s["qsl"] = _long([sum(counts[:i]) for i in range(len(counts) + 1)])
        s["max_q"] = max(counts)
        s["ancestors"] = _ancestor_words(counts, seed)
        s["q"] = rand(sum(counts), hq, d)
    else:
        lens = _lengths(case["batch"], case["ctx_lo"], case["ctx_hi"], 1)
        s["q"] = rand(len(lens), hq, d) if kind in ("weigh", "sparse") else None
    tables, blocks = _tables(lens, seed)
    s["bt"], s["ctx"], s["max_ctx"] = _padded(tables), _long(lens), max(lens)
    s["k"], s["v"] = rand(blocks, BLOCK, hkv, d), rand(blocks, BLOCK, hkv, d)
    if kind == "move":
        counts = _kept_counts(case)
        s["start"] = _long([n - case["drafted"] for n in lens]) if case["drafted"] else None
        first = s["ctx"] - case["drafted"] if case["drafted"] else torch.zeros_like(s["ctx"])
        span = s["ctx"] - first
        # For each list, `counts` different positions of its span, in order.
        lists = (len(lens), hkv) if case["per_head"] else (len(lens), 1)
        noise = torch.rand(*lists, int(span.max()), generator=gen, device=DEVICE)
        at = torch.arange(noise.shape[-1], device=DEVICE)
        noise = noise.masked_fill(at >= span[:, None, None], 2.0)
        picked = noise.argsort(-1)[..., :max(counts)]
        column = torch.arange(max(counts), device=DEVICE)
        absent = column >= _long(counts)[:, None, None]
        big = 1 << 40
        kept = (picked + first[:, None, None]).masked_fill(absent, big).sort(-1).values
        kept = kept.masked_fill(kept == big, -1)
        s["kept"] = kept if case["per_head"] else kept[:, 0].contiguous()
    if kind in ("weigh", "evict"):
        # What some hundred steps have added: a few heavy keys, many light ones.
        s["weights"] = torch.empty(blocks, hkv, BLOCK, device=DEVICE).exponential_(generator=gen)
        s["weights"] = s["weights"] ** 2 * 0.3
    if kind == "bounds":
        s["bounds"] = rand(blocks, 2, hkv, d)
        s["starts"] = _long(_starts(case, lens)) if case["new"] else None
    if kind == "sparse":
        s["bounds"] = torch.stack([s["k"].amin(1), s["k"].amax(1)], dim=1)
    return s


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------
def _keys(cache, tables, count):
    """The first `count` rows of each table's blocks: [S, Hkv, count, D] in 32 bits."""
    hkv, d = cache.shape[2:]
    rows = cache[tables.clamp(min=0)].view(tables.shape[0], -1, hkv, d)[:, :count]
    return rows.float().transpose(1, 2).contiguous()


def _scores(s, q, k):
    """Scores of q [S, Hq, L, D] on k [S, Hkv, N, D]: [S, Hq, L, N]."""
    seqs, hq, length, d = q.shape
    hkv = k.shape[1]
    q = q.reshape(seqs, hkv, hq // hkv * length, d)
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()).view(seqs, hq, length, -1) * s["scale"]
    cap = s["case"]["cap"]
    return cap * torch.tanh(x / cap) if cap > 0 else x


def _values(p, v):
    """p [S, Hq, L, N] times v [S, Hkv, N, D]: [S, Hq, L, D]."""
    seqs, hq, length, n = p.shape
    hkv = v.shape[1]
    return torch.matmul(p.reshape(seqs, hkv, hq // hkv * length, n), v).view(seqs, hq, length, -1)


def _softmax(x, visible):
    x = x.masked_fill(~visible, float("-inf"))
    p = (x - x.amax(-1, keepdim=True)).exp()
    return p / p.sum(-1, keepdim=True)


def _plain_tree(s):
    q, ctx, qsl = s["q"], s["ctx"], s["qsl"]
    lens = qsl[1:] - qsl[:-1]
    row = torch.arange(s["max_q"], device=q.device)
    token = (qsl[:-1, None] + row).clamp(max=q.shape[0] - 1)
    padded = q[token].float().transpose(1, 2)
    k, v = _keys(s["k"], s["bt"], s["max_ctx"]), _keys(s["v"], s["bt"], s["max_ctx"])
    # Place of a key among the drafted ones; below 0 it is an older one.
    node = torch.arange(s["max_ctx"], device=q.device)[None] - (ctx - lens)[:, None]
    at = node.clamp(min=0, max=64 * s["ancestors"].shape[1] - 1)
    words = torch.gather(s["ancestors"][token], 2,
                         (at // 64)[:, None].expand(-1, s["max_q"], -1))
    bit = (words >> (at % 64)[:, None]) & 1
    visible = (node[:, None] < 0) | ((bit != 0) & (node < lens[:, None])[:, None])
    # Rows of padding see the first key, so that they have a maximum.
    visible = visible | ((row[None, :, None] >= lens[:, None, None]) & (node == node[:, :1])[:, None])
    p = _softmax(_scores(s, padded, k), visible[:, None])
    out = _values(p, v).transpose(1, 2)  # [S, L, Hq, D]
    every = torch.arange(q.shape[0], device=q.device)
    owner = torch.searchsorted(qsl[1:].contiguous(), every, right=True)
    return out[owner, every - qsl[owner]].to(q.dtype)


def _slots(s, positions):
    """Slots [B, Hkv, n] of positions [B, Hkv, n]."""
    batch = positions.shape[0]
    block = torch.gather(s["bt"], 1, (positions // BLOCK).view(batch, -1)).view_as(positions)
    return block * BLOCK + positions % BLOCK


def _move(s, kept, start):
    """Rows start + i <- kept[i] for lists kept [B, Hkv, n], -1 past their ends."""
    hkv, d = s["k"].shape[2:]
    count = (kept >= 0).sum(-1, keepdim=True)
    # Past its end a list repeats its last move.
    i = torch.minimum(torch.arange(kept.shape[-1], device=kept.device), count - 1)
    src = _slots(s, torch.gather(kept, 2, i))
    dst = _slots(s, i + start[:, None, None])
    head = torch.arange(hkv, device=kept.device)[None, :, None]
    for name in ("k", "v"):
        rows = s[name].view(-1, hkv, d)
        rows[dst, head] = rows[src, head]
    if "weights" in s:
        w = s["weights"]
        w[dst // BLOCK, head, dst % BLOCK] = w[src // BLOCK, head, src % BLOCK]


def _plain_move(s):
    hkv = s["k"].shape[2]
    kept = s["kept"] if s["kept"].ndim == 3 else s["kept"][:, None].expand(-1, hkv, -1)
    _move(s, kept, torch.zeros_like(s["ctx"]) if s["start"] is None else s["start"])
    return s["k"], s["v"]


def _plain_weigh(s):
    q, ctx = s["q"], s["ctx"]
    batch, hq, _ = q.shape
    hkv = s["k"].shape[2]
    k, v = _keys(s["k"], s["bt"], s["max_ctx"]), _keys(s["v"], s["bt"], s["max_ctx"])
    key = torch.arange(s["max_ctx"], device=q.device)
    visible = key < ctx[:, None]
    p = _softmax(_scores(s, q.float()[:, :, None], k), visible[:, None, None])
    out = _values(p, v)[:, :, 0].to(q.dtype)
    w = p[:, :, 0].view(batch, hkv, hq // hkv, -1).sum(2)
    # Positions past a request's end repeat its newest key's.
    at = torch.minimum(key[None, None], ctx[:, None, None] - 1).expand(batch, hkv, -1)
    slot = _slots(s, at)
    head = torch.arange(hkv, device=q.device)[None, :, None]
    before = s["weights"][slot // BLOCK, head, slot % BLOCK]
    before = before.masked_fill((at == ctx[:, None, None] - 1), 0.0)
    s["weights"][slot // BLOCK, head, slot % BLOCK] = before + torch.gather(w, 2, at)
    return out, s["weights"]


def _best(score, forced, exists, budget):
    """Of each row the `budget` first places: the forced, then the best scores,
    ties by place; ascending, -1 past the end."""
    n = score.shape[-1]
    place = torch.arange(n, device=score.device).expand_as(score)
    _, order = torch.sort(score, dim=-1, descending=True, stable=True)
    rank = torch.where(exists, torch.where(forced, 0, 1), 2).expand_as(score)
    _, by = torch.sort(torch.gather(rank, -1, order), dim=-1, stable=True)
    order = torch.gather(order, -1, by)[..., :budget]
    kept = torch.where(torch.gather(exists.expand_as(score), -1, order),
                       torch.gather(place, -1, order), n).sort(-1).values
    kept = kept.masked_fill(kept == n, -1)
    return torch.nn.functional.pad(kept, (0, budget - kept.shape[-1]), value=-1)


def _plain_evict(s):
    case, ctx = s["case"], s["ctx"]
    hkv = s["k"].shape[2]
    at = torch.arange(s["max_ctx"], device=DEVICE)[None, None]
    exists = at < ctx[:, None, None]
    slot = _slots(s, torch.minimum(at, ctx[:, None, None] - 1).expand(-1, hkv, -1))
    head = torch.arange(hkv, device=DEVICE)[None, :, None]
    w = s["weights"][slot // BLOCK, head, slot % BLOCK]
    forced = (at < case["sinks"]) | (at >= ctx[:, None, None] - case["recent"])
    kept = _best(w, forced, exists, case["budget"])
    _move(s, kept, torch.zeros_like(ctx))
    return kept, ctx.clamp(max=case["budget"]), s["k"], s["v"], s["weights"]


def _plain_bounds(s):
    ctx = s["ctx"]
    starts = torch.zeros_like(ctx) if s["starts"] is None else s["starts"]
    block = torch.arange(s["bt"].shape[1], device=DEVICE)[None]
    changed = (block >= (starts // BLOCK)[:, None]) & (block * BLOCK < ctx[:, None])
    position = block[..., None] * BLOCK + torch.arange(BLOCK, device=DEVICE)
    k = s["k"][s["bt"].clamp(min=0)].float()  # [B, W, BLOCK, Hkv, D]
    absent = (position >= ctx[:, None, None])[..., None, None]
    low = k.masked_fill(absent, float("inf")).amin(2)
    high = k.masked_fill(absent, float("-inf")).amax(2)
    new = torch.stack([low, high], dim=2).to(s["k"].dtype)
    # Blocks that are not changed, or not there, write to a row behind the last.
    where = torch.where(changed, s["bt"], s["bounds"].shape[0])
    wide = torch.cat([s["bounds"], s["bounds"][:1]])
    wide[where] = new
    s["bounds"].copy_(wide[:-1])
    return s["bounds"]


def _plain_sparse(s):
    case, q, ctx = s["case"], s["q"], s["ctx"]
    batch, hq, d = q.shape
    hkv = s["k"].shape[2]
    blocks = (ctx + BLOCK - 1) // BLOCK
    at = torch.arange(s["bt"].shape[1], device=DEVICE)[None, None]
    bound = s["bounds"][s["bt"].clamp(min=0)].double()  # [B, W, 2, Hkv, D]
    low = bound[:, :, 0].permute(0, 2, 3, 1).contiguous()
    high = bound[:, :, 1].permute(0, 2, 3, 1).contiguous()
    x = q.double().view(batch, hkv, hq // hkv, d)
    # The larger of q * low and q * high, element by element.
    score = torch.matmul(x.clamp(min=0), high) + torch.matmul(x.clamp(max=0), low)
    n = blocks[:, None, None]
    forced = (at < case["sinks"]) | (at >= n - case["recent"])
    chosen = _best(score.amax(2), forced, at < n, case["budget"])
    block = torch.gather(s["bt"], 1, chosen.clamp(min=0).view(batch, -1)).view_as(chosen)
    head = torch.arange(hkv, device=DEVICE)[None, :, None, None]
    offset = torch.arange(BLOCK, device=DEVICE)
    k = s["k"][block[..., None], offset, head].float().view(batch, hkv, -1, d)
    v = s["v"][block[..., None], offset, head].float().view(batch, hkv, -1, d)
    position = chosen[..., None] * BLOCK + offset
    visible = (chosen[..., None] >= 0) & (position < ctx[:, None, None, None])
    visible = visible.view(batch, hkv, 1, 1, -1).expand(-1, -1, hq // hkv, -1, -1)
    p = _softmax(_scores(s, q.float()[:, :, None], k),
                 visible.reshape(batch, hq, 1, visible.shape[-1]))
    return _values(p, v)[:, :, 0].to(q.dtype), chosen


# ---------------------------------------------------------------------------
# The framework's own
# ---------------------------------------------------------------------------
_own = {}


def _calls():
    if not _own:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        sys.path.insert(1, os.path.join(root, "mini-llm-runtime_amd"))
        from mini_llm_runtime_amd.kernels import key_eviction, sparse_attention, tree_attention

        _own.update(tree=tree_attention.paged_attention_tree, move=key_eviction.compact_keys,
                    weigh=key_eviction.paged_attention_decode_weighted,
                    evict=key_eviction.evict_keys, bounds=sparse_attention.update_key_bounds,
                    sparse=sparse_attention.paged_attention_decode_sparse)
    return _own


def _run_own(s):
    case = s["case"]
    kind = case["kind"]
    call = _calls()[kind]
    # The step's metadata is checked once a step, not in every layer.
    if kind == "tree":
        return call(s["q"], s["k"], s["v"], s["bt"], s["qsl"], s["ctx"], s["ancestors"], BLOCK,
                    softcap=case["cap"], scale=s["scale"], max_query_len=s["max_q"],
                    validate=False)
    if kind == "move":
        call(s["k"], s["v"], s["bt"], s["kept"], BLOCK, start=s["start"], validate=False)
        return s["k"], s["v"]
    if kind == "weigh":
        out = call(s["q"], s["k"], s["v"], s["weights"], s["bt"], s["ctx"], BLOCK,
                   softcap=case["cap"], scale=s["scale"], validate=False)
        return out, s["weights"]
    if kind == "evict":
        kept, lens = call(s["k"], s["v"], s["weights"], s["bt"], s["ctx"], BLOCK, case["budget"],
                          sinks=case["sinks"], recent=case["recent"], validate=False)
        return kept, lens, s["k"], s["v"], s["weights"]
    if kind == "bounds":
        call(s["k"], s["bounds"], s["bt"], s["ctx"], BLOCK, starts=s["starts"],
             max_new=case["new"] or None, validate=False)
        return s["bounds"]
    return call(s["q"], s["k"], s["v"], s["bounds"], s["bt"], s["ctx"], BLOCK, case["budget"],
                sinks=case["sinks"], recent=case["recent"], softcap=case["cap"],
                scale=s["scale"], return_blocks=True, validate=False)


_PLAIN = {"tree": _plain_tree, "move": _plain_move, "weigh": _plain_weigh, "evict": _plain_evict,
          "bounds": _plain_bounds, "sparse": _plain_sparse}


def run(s):
    if own:
        return _run_own(s)
    return _PLAIN[s["case"]["kind"]](s)


# ---------------------------------------------------------------------------
# The definitions in 64 bits, request by request
# ---------------------------------------------------------------------------
def _rows_of(s, i, positions):
    """Slots of request i's positions."""
    return s["bt"][i][positions // BLOCK] * BLOCK + positions % BLOCK


def _weights_of(s, q, k, seen):
    """Attention weights of one head: q [n, D] over keys k [N, D] where seen [n, N]."""
    x = q.double() @ k.double().T.contiguous() * s["scale"]
    if s["case"]["cap"]:
        x = torch.tanh(x / s["case"]["cap"]) * s["case"]["cap"]
    return torch.softmax(torch.where(seen, x, -math.inf), -1)


def _exact_tree(s):
    hq, hkv, d = (s["case"][n] for n in ("hq", "hkv", "d"))
    k, v = s["k"].view(-1, hkv, d), s["v"].view(-1, hkv, d)
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE)
    first = s["qsl"].tolist()
    for i, n in enumerate(s["ctx"].tolist()):
        rows = slice(first[i], first[i + 1])
        count = first[i + 1] - first[i]
        seen = torch.ones(count, n, dtype=torch.bool, device=DEVICE)
        for j in range(count):
            seen[:, n - count + j] = (s["ancestors"][rows, j // 64] >> j % 64) % 2 == 1
        slot = _rows_of(s, i, torch.arange(n, device=DEVICE))
        for h in range(hq):
            p = _weights_of(s, s["q"][rows, h], k[slot, h * hkv // hq], seen)
            out[rows, h] = p @ v[slot, h * hkv // hq].double()
    return out


def _exact_move(s, lists, starts, to):
    """Copies by list (per KV head or for all) from the state's tensors to `to`."""
    hkv, d = s["k"].shape[2:]
    for i, start in enumerate(starts):
        for h in range(hkv):
            kept = lists[i][h if lists.ndim == 3 else slice(None)]
            kept = kept[kept >= 0]
            src = _rows_of(s, i, kept)
            dst = _rows_of(s, i, start + torch.arange(len(kept), device=DEVICE))
            for name in ("k", "v"):
                to[name].view(-1, hkv, d)[dst, h] = s[name].view(-1, hkv, d)[src, h].double()
            if "weights" in to:
                to["weights"][dst // BLOCK, h, dst % BLOCK] = (
                    s["weights"][src // BLOCK, h, src % BLOCK].double())


def _exact_weigh(s):
    hq, hkv, d = (s["case"][n] for n in ("hq", "hkv", "d"))
    k, v = s["k"].view(-1, hkv, d), s["v"].view(-1, hkv, d)
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE)
    total = s["weights"].double()
    for i, n in enumerate(s["ctx"].tolist()):
        slot = _rows_of(s, i, torch.arange(n, device=DEVICE))
        total[slot[-1] // BLOCK, :, slot[-1] % BLOCK] = 0
        for h in range(hq):
            g = h * hkv // hq
            p = _weights_of(s, s["q"][i, h][None], k[slot, g], slot[None] >= 0)[0]
            out[i, h] = p @ v[slot, g].double()
            total[slot // BLOCK, g, slot % BLOCK] += p
    return out, total


def _first_by(score, count):
    """The places of the `count` largest, ties by place, ascending."""
    return torch.argsort(-score, stable=True)[:max(count, 0)].sort().values


def _exact_choice(score, sinks, recent, budget):
    """score [n]: what stays of n places."""
    n = score.shape[0]
    if n <= budget:
        return torch.arange(n, device=DEVICE)
    head, tail = torch.arange(sinks, device=DEVICE), torch.arange(n - recent, n, device=DEVICE)
    middle = sinks + _first_by(score[sinks:n - recent], budget - sinks - recent)
    return torch.cat([head, middle, tail])


def _exact_evict(s):
    case, hkv = s["case"], s["k"].shape[2]
    kept = torch.full((case["batch"], hkv, case["budget"]), -1, dtype=torch.long, device=DEVICE)
    lens = s["ctx"].tolist()
    for i, n in enumerate(lens):
        slot = _rows_of(s, i, torch.arange(n, device=DEVICE))
        for h in range(hkv):
            w = s["weights"][slot // BLOCK, h, slot % BLOCK].double()
            at = _exact_choice(w, case["sinks"], case["recent"], case["budget"])
            kept[i, h, :len(at)] = at
    to = {name: s[name].double() for name in ("k", "v", "weights")}
    _exact_move(s, kept, [0] * len(lens), to)
    return (kept, _long([min(n, case["budget"]) for n in lens]), to["k"], to["v"], to["weights"])


def _exact_bounds(s):
    out = s["bounds"].double()
    lens = s["ctx"].tolist()
    starts = [0] * len(lens) if s["starts"] is None else s["starts"].tolist()
    hkv, d = s["k"].shape[2:]
    for i, n in enumerate(lens):
        whole = torch.arange(starts[i] // BLOCK, n // BLOCK, device=DEVICE)
        block = s["bt"][i][whole]
        k = s["k"][block].double()
        out[block, 0], out[block, 1] = k.amin(1), k.amax(1)
        if n % BLOCK:
            block = s["bt"][i][n // BLOCK]
            k = s["k"][block, :n % BLOCK].double()
            out[block, 0], out[block, 1] = k.amin(0), k.amax(0)
    return out


def _exact_sparse(s):
    case = s["case"]
    hq, hkv, d = (case[n] for n in ("hq", "hkv", "d"))
    group = hq // hkv
    k, v = s["k"].view(-1, hkv, d), s["v"].view(-1, hkv, d)
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE)
    chosen = torch.full((case["batch"], hkv, case["budget"]), -1, dtype=torch.long, device=DEVICE)
    for i, n in enumerate(s["ctx"].tolist()):
        table = s["bt"][i][:-(-n // BLOCK)]
        for g in range(hkv):
            score = torch.full((len(table),), -math.inf, dtype=torch.float64, device=DEVICE)
            low, high = s["bounds"][table, 0, g].double(), s["bounds"][table, 1, g].double()
            for h in range(g * group, (g + 1) * group):
                x = s["q"][i, h].double()
                score = torch.maximum(score, torch.maximum(low * x, high * x).sum(-1))
            at = _exact_choice(score, case["sinks"], case["recent"], case["budget"])
            chosen[i, g, :len(at)] = at
            position = (at[:, None] * BLOCK + torch.arange(BLOCK, device=DEVICE)).flatten()
            slot = _rows_of(s, i, position[position < n])
            for h in range(g * group, (g + 1) * group):
                p = _weights_of(s, s["q"][i, h][None], k[slot, g], slot[None] >= 0)
                out[i, h] = (p @ v[slot, g].double())[0]
    return out, chosen


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "move":
        to = {name: s[name].double() for name in ("k", "v")}
        starts = [0] * case["batch"] if s["start"] is None else s["start"].tolist()
        _exact_move(s, s["kept"], starts, to)
        return to["k"], to["v"]
    return {"tree": _exact_tree, "weigh": _exact_weigh, "evict": _exact_evict,
            "bounds": _exact_bounds, "sparse": _exact_sparse}[case["kind"]](s)
