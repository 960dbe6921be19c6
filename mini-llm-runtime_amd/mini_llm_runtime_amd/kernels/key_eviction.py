"""Which keys a paged cache holds on to (csrc/key_eviction.hip). No reference
counterpart; beside the plain calls of ``paged_attention``, with the same caches and tables.

``paged_attention_decode_weighted`` decodes a step and adds up what attention each key
gets. ``evict_keys`` keeps, for each KV head, the first keys, the last ones and the
heaviest of the others, and moves them together in place, so that the blocks behind
them can be freed. ``compact_keys`` is the move alone, by given lists: the accepted path
of drafted tokens, or a choice of the caller's own.

The sums are FP32, laid out like the cache with positions last: key_weights
[num_blocks, Hkv, block_size]. A step sets its newest key's entry; the entries of a
prompt's keys, which no step has set, are the caller's to clear. The decode's numbers are
those of ``tree_attention``: FP32 sums, one rounding of the result.
"""

from __future__ import annotations

import torch

from .. import _lib
from .paged_attention import _as_index_tensor, _check_cache_pair, _validate_tables
from .scored_attention import _aligned_q, _check, _out, _table, _workspace

_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def _check_weights(key_weights: torch.Tensor, k_cache: torch.Tensor) -> None:
    num_blocks, block_size, num_kv_heads, _ = k_cache.shape
    if (key_weights.shape != (num_blocks, num_kv_heads, block_size)
            or key_weights.dtype != torch.float32 or not key_weights.is_contiguous()):
        raise ValueError("key_weights must be a contiguous FP32 tensor of shape "
                         "[num_blocks, Hkv, block_size]")


def _check_cache(k_cache, v_cache, block_size, what, *more) -> torch.device:
    _check_cache_pair(k_cache, v_cache)
    _, cache_block, _, head_dim = k_cache.shape
    if block_size != cache_block:
        raise ValueError("block_size does not match KV cache layout")
    dtype = k_cache.dtype
    if dtype not in _DTYPES:
        raise TypeError(f"{what}: unsupported dtype {dtype}")
    if v_cache.dtype != dtype:
        raise TypeError(f"{what}: k_cache and v_cache must share one dtype")
    if head_dim * k_cache.element_size() % 16 or not 0 < head_dim <= 1024:
        raise ValueError(f"{what} takes head_dim in multiples of 16 bytes, up to 1024 elements")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError(f"{what}: k_cache and v_cache must be contiguous block pools")
    return _lib.require_hip(k_cache, v_cache, *more, what=what)


def _shared(block_tables: torch.Tensor, first: torch.Tensor, end: torch.Tensor) -> torch.Tensor:
    """Whether a block stands twice in the columns [first, end) of the tables."""
    column = torch.arange(block_tables.shape[1], device=block_tables.device)[None, :]
    used = (column >= first[:, None]) & (column < end[:, None])
    ids = torch.where(used, block_tables, -1).flatten().sort().values
    return ((ids[1:] == ids[:-1]) & (ids[1:] >= 0)).any()


def _newest_is_shared(block_tables: torch.Tensor, seq_lens: torch.Tensor,
                      block_size: int) -> torch.Tensor:
    """Whether a request's newest key, in a block that it fills to `fill` keys, is a key of
    another place in the tables too: whether the same block is filled as far there."""
    column = torch.arange(block_tables.shape[1], device=block_tables.device)[None, :]
    last = torch.div(seq_lens - 1, block_size, rounding_mode="floor")[:, None]
    fill = (seq_lens[:, None] - column * block_size).clamp(max=block_size)
    # By block, then by fill, and of those that fill alike the newest keys' first: such a
    # place must have no other of its block behind it.
    order = 2 * (block_tables * (block_size + 1) + fill) + (column != last)
    order = torch.where(column <= last, order, -1).flatten().sort().values
    block = torch.div(order, 2 * (block_size + 1), rounding_mode="floor")
    return ((order[:-1] >= 0) & (order[:-1] % 2 == 0) & (block[1:] == block[:-1])).any()


def paged_attention_decode_weighted(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    key_weights: torch.Tensor,
    block_tables: torch.Tensor,
    seq_lens: torch.Tensor,
    block_size: int,
    *,
    softcap: float = 0.0,
    scale: float | None = None,
    validate: bool = True,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """paged_attention_decode_scored (without a bias) that also adds each key's attention
    weight, summed over the query heads of its KV head, to key_weights in place. The entry
    of a request's newest key, at position seq_lens[b] - 1, is set, whatever it held. With
    validate=False a seq_lens of 0 (a padded row) gives zeros and adds nothing.

    Requests may share blocks, but no request's newest key may be another's key too, which
    validate=True checks with the tables: each adds to the entries of the shared keys, in
    no particular order, so that the last bits of such a sum may differ from run to run.
    The workspace holds the scores of the batch: 4 bytes for every query head and every
    position that the tables cover.
    """
    what = "paged_attention_decode_weighted"
    device, _ = _check(q, k_cache, v_cache, block_size, softcap, None, what)
    _check_weights(key_weights, k_cache)
    if key_weights.device != device:
        raise RuntimeError(f"{what}: operands are on different devices")
    batch, num_q_heads, head_dim = q.shape
    block_tables = _table(block_tables, batch, device)
    seq_lens = _as_index_tensor(seq_lens, device).contiguous()
    if seq_lens.shape != (batch,):
        raise ValueError("seq_lens length must match batch size of q")
    out = _out(q, out, device)
    if batch == 0:
        return out
    num_blocks, _, num_kv_heads, _ = k_cache.shape
    if validate:
        _validate_tables(block_tables, seq_lens, block_size, num_blocks)
        if _newest_is_shared(block_tables, seq_lens, block_size):
            raise ValueError("a request's newest key must be no other key too")
    q = _aligned_q(q)
    width = block_tables.shape[1]
    lib = _lib.load()
    with _lib.on(device):
        nbytes = lib.mlr_paged_decode_weighted_workspace_size(
            batch, num_q_heads, num_kv_heads, head_dim, width * block_size)
        ws = _workspace(nbytes, device)
        status = lib.mlr_paged_decode_weighted(
            q.data_ptr(), q.stride(0), q.stride(1), k_cache.data_ptr(), v_cache.data_ptr(),
            key_weights.data_ptr(), num_blocks, block_size, num_kv_heads, head_dim,
            block_tables.data_ptr(), block_tables.stride(0), width, seq_lens.data_ptr(), batch,
            num_q_heads, head_dim ** -0.5 if scale is None else scale, softcap,
            _lib.DTYPE_CODES[q.dtype], None if ws is None else ws.data_ptr(), nbytes,
            out.data_ptr(), out.stride(0), out.stride(1), _lib.stream_handle(device))
    _lib.check(status, "mlr_paged_decode_weighted")
    return out


def evict_keys(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    key_weights: torch.Tensor,
    block_tables: torch.Tensor,
    seq_lens: torch.Tensor,
    block_size: int,
    budget: int,
    *,
    sinks: int = 4,
    recent: int | None = None,
    validate: bool = True,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Cuts each request to `budget` keys for each KV head: its first `sinks`, its last
    `recent` (None: half the budget, or what the sinks leave of it) and the heaviest of the
    others by key_weights (ties: the lower position; NaN counts as -infinity). `budget` is
    at least `sinks` and `recent` together. What stays keeps its order and moves,
    with its key_weights, to the positions 0, 1, ... of the request, in place; what lies
    behind is left as it is. With validate=False a seq_lens of 0 (a padded row) keeps none.

    Returns (kept, new_lens): int64 [B, Hkv, budget], the positions that stayed, -1 past
    the end, and int64 [B], min(seq_lens, budget). A request no longer than the budget
    is not changed. Requests must not share blocks, which validate=True checks with the
    tables.
    """
    what = "evict_keys"
    device = _check_cache(k_cache, v_cache, block_size, what, key_weights)
    _check_weights(key_weights, k_cache)
    if recent is None:
        recent = max(min(budget // 2, budget - sinks), 0)
    if sinks < 0 or recent < 0 or budget < sinks + recent:
        raise ValueError("budget must be at least sinks + recent, and none of them negative")
    if not 0 <= budget < 1 << 31:
        raise ValueError("budget must be below 2^31")
    seq_lens = _as_index_tensor(seq_lens, device).contiguous()
    if seq_lens.ndim != 1:
        raise ValueError("seq_lens must have shape [B]")
    batch = seq_lens.shape[0]
    block_tables = _table(block_tables, batch, device)
    num_blocks, _, num_kv_heads, head_dim = k_cache.shape
    if validate and batch:
        _validate_tables(block_tables, seq_lens, block_size, num_blocks)
        end = torch.div(seq_lens + (block_size - 1), block_size, rounding_mode="floor")
        if _shared(block_tables, torch.zeros_like(end), end):
            raise ValueError("requests that share a block cannot be cut")
    kept = torch.empty(batch, num_kv_heads, budget, dtype=torch.long, device=device)
    new_lens = torch.empty(batch, dtype=torch.long, device=device)
    with _lib.on(device):
        status = _lib.load().mlr_evict_keys(
            k_cache.data_ptr(), v_cache.data_ptr(), key_weights.data_ptr(), num_blocks, block_size,
            num_kv_heads, head_dim, block_tables.data_ptr(), block_tables.stride(0),
            block_tables.shape[1], seq_lens.data_ptr(), batch, budget, sinks, recent,
            _lib.DTYPE_CODES[k_cache.dtype], kept.data_ptr(), new_lens.data_ptr(),
            _lib.stream_handle(device))
    _lib.check(status, "mlr_evict_keys")
    return kept, new_lens


def compact_keys(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_tables: torch.Tensor,
    kept: torch.Tensor,
    block_size: int,
    *,
    start: torch.Tensor | None = None,
    key_weights: torch.Tensor | None = None,
    validate: bool = True,
) -> None:
    """Moves cache rows together, in place: the row at position kept[b, h, i] of request b
    and KV head h goes to position start[b] + i (start None: 0), and its key_weights
    entry, if given, with it. kept is int64 [B, Hkv, n], or [B, n] for all KV heads alike;
    a list ascends from start[b] on, -1 past its end. What lies behind the last row is left
    as it is.

    Of a drafted tree that was verified, start is the length before it and kept the
    positions of the accepted path. Requests must not share the blocks from start on to
    their last kept position; validate=True checks that, the lists and the tables.
    """
    what = "compact_keys"
    device = _check_cache(k_cache, v_cache, block_size, what,
                          *(() if key_weights is None else (key_weights,)))
    if key_weights is not None:
        _check_weights(key_weights, k_cache)
    num_blocks, _, num_kv_heads, head_dim = k_cache.shape
    kept = _as_index_tensor(kept, device)
    if kept.ndim not in (2, 3) or (kept.ndim == 3 and kept.shape[1] != num_kv_heads):
        raise ValueError("kept must have shape [B, n] or [B, Hkv, n]")
    if kept.numel() and kept.stride(-1) != 1:
        kept = kept.contiguous()
    batch, num_kept = kept.shape[0], kept.shape[-1]
    block_tables = _table(block_tables, batch, device)
    if start is not None:
        start = _as_index_tensor(start, device).contiguous()
        if start.shape != (batch,):
            raise ValueError("start must hold one position per request")
    if batch == 0 or num_kept == 0:
        return
    if validate:
        _validate_lists(block_tables, kept, start, block_size, num_blocks)
    with _lib.on(device):
        status = _lib.load().mlr_compact_keys(
            k_cache.data_ptr(), v_cache.data_ptr(),
            None if key_weights is None else key_weights.data_ptr(), num_blocks, block_size,
            num_kv_heads, head_dim, block_tables.data_ptr(), block_tables.stride(0),
            block_tables.shape[1], kept.data_ptr(), kept.stride(0),
            kept.stride(1) if kept.ndim == 3 else 0, num_kept,
            None if start is None else start.data_ptr(), batch,
            _lib.DTYPE_CODES[k_cache.dtype], _lib.stream_handle(device))
    _lib.check(status, "mlr_compact_keys")


def _validate_lists(block_tables, kept, start, block_size, num_blocks) -> None:
    """One host sync for the checks of compact_keys' lists and tables."""
    lists = kept if kept.ndim == 3 else kept[:, None]
    first = torch.zeros_like(lists[:, 0, 0]) if start is None else start
    there = lists >= 0
    to = first[:, None, None] + torch.arange(lists.shape[-1], device=lists.device)
    last = lists.amax((1, 2))  # -1: nothing to move
    column = torch.arange(block_tables.shape[1], device=lists.device)[None, :]
    low = torch.div(first.clamp(min=0), block_size, rounding_mode="floor")
    end = torch.div(last, block_size, rounding_mode="floor") + 1
    end = torch.where(last >= 0, end, 0)
    used = (column >= low[:, None]) & (column < end[:, None])
    flags = torch.stack([
        (first < 0).any(),
        (there[..., 1:] & ~(there[..., :-1] & (lists[..., 1:] > lists[..., :-1]))).any(),
        (there & (lists < to)).any(),
        (end > block_tables.shape[1]).any(),
        (used & ((block_tables < 0) | (block_tables >= num_blocks))).any(),
        _shared(block_tables, low, end)]).tolist()
    for flag, message in zip(flags, (
            "start must not be negative",
            "kept must ascend, with -1 only past a list's end",
            "kept[..., i] must be at least start + i",
            "block_tables do not contain enough blocks for the kept positions",
            "block_tables contain an invalid physical block",
            "requests that share a block cannot be compacted there")):
        if flag:
            raise ValueError(message)
