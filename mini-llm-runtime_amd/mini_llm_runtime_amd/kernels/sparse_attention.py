"""Decode over the blocks of a long cache that a cheap score selects
(csrc/sparse_attention.hip, csrc/scored_rows.hip). No reference counterpart; beside the plain
calls of ``paged_attention``, with the same caches and tables.

``update_key_bounds`` keeps, for each block and KV head, the elementwise minimum and maximum
of its keys: key_bounds [num_blocks, 2, Hkv, D], in the cache's type.
``paged_attention_decode_sparse`` scores each block by the largest q.k that keys within
its bounds could have and attends to the keys of the best blocks: of a long context
it reads the bounds and `budget` blocks instead of all keys and values. Its numbers are
those of ``tree_attention``: FP32 sums, one rounding of the result.
"""

from __future__ import annotations

import torch

from .. import _lib
from .paged_attention import _as_index_tensor, _validate_tables
from .scored_attention import _aligned_q, _check, _out, _table, _workspace


def _check_bounds(key_bounds: torch.Tensor, k_cache: torch.Tensor) -> None:
    num_blocks, _, num_kv_heads, head_dim = k_cache.shape
    if (key_bounds.shape != (num_blocks, 2, num_kv_heads, head_dim)
            or key_bounds.dtype != k_cache.dtype or not key_bounds.is_contiguous()):
        raise ValueError("key_bounds must be a contiguous tensor of shape "
                         "[num_blocks, 2, Hkv, D] in the cache's dtype")


def update_key_bounds(
    k_cache: torch.Tensor,
    key_bounds: torch.Tensor,
    block_tables: torch.Tensor,
    seq_lens: torch.Tensor,
    block_size: int,
    *,
    starts: torch.Tensor | None = None,
    max_new: int | None = None,
    validate: bool = True,
) -> None:
    """Writes the bounds of each block that holds a position of [starts[b], seq_lens[b])
    (starts None: of every block of the request) from its keys, in place. A NaN among
    them gives NaN.

    After a step that appended one token a request: starts = seq_lens - 1, max_new = 1.
    max_new, at least the longest such range, sizes the launch of a call with starts; without
    it the tables' width does. Full blocks that requests share are written by each, with the
    same values; the bounds of a shared block that one of them fills further than another
    may be either's.
    """
    what = "update_key_bounds"
    if k_cache.ndim != 4:
        raise ValueError("k_cache must have shape [num_blocks, block_size, Hkv, D]")
    num_blocks, cache_block, num_kv_heads, head_dim = k_cache.shape
    if block_size != cache_block:
        raise ValueError("block_size does not match KV cache layout")
    if k_cache.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise TypeError(f"{what}: unsupported dtype {k_cache.dtype}")
    if head_dim * k_cache.element_size() % 16 or not 0 < head_dim <= 1024:
        raise ValueError(f"{what} takes head_dim in multiples of 16 bytes, up to 1024 elements")
    if not k_cache.is_contiguous():
        raise ValueError(f"{what}: k_cache must be a contiguous block pool")
    _check_bounds(key_bounds, k_cache)
    device = _lib.require_hip(k_cache, key_bounds, what=what)
    seq_lens = _as_index_tensor(seq_lens, device).contiguous()
    if seq_lens.ndim != 1:
        raise ValueError("seq_lens must have shape [B]")
    batch = seq_lens.shape[0]
    block_tables = _table(block_tables, batch, device)
    if starts is not None:
        starts = _as_index_tensor(starts, device).contiguous()
        if starts.shape != (batch,):
            raise ValueError("starts must hold one position per request")
    width = block_tables.shape[1]
    if max_new is not None and max_new < 0:
        raise ValueError("max_new cannot be negative")
    max_new = width * block_size if max_new is None else min(max_new, width * block_size)
    if batch == 0:
        return
    if validate:
        _validate_tables(block_tables, seq_lens, block_size, num_blocks)
        if starts is not None:
            low, many = torch.stack([(starts < 0).any(),
                                     (seq_lens - starts > max_new).any()]).tolist()
            if low:
                raise ValueError("starts must not be negative")
            if many:
                raise ValueError("max_new must cover the longest range of new positions")
    with _lib.on(device):
        status = _lib.load().mlr_update_key_bounds(
            k_cache.data_ptr(), key_bounds.data_ptr(), num_blocks, block_size, num_kv_heads,
            head_dim, block_tables.data_ptr(), block_tables.stride(0), width,
            seq_lens.data_ptr(), None if starts is None else starts.data_ptr(), max_new, batch,
            _lib.DTYPE_CODES[k_cache.dtype], _lib.stream_handle(device))
    _lib.check(status, "mlr_update_key_bounds")


def paged_attention_decode_sparse(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    key_bounds: torch.Tensor,
    block_tables: torch.Tensor,
    seq_lens: torch.Tensor,
    block_size: int,
    budget: int,
    *,
    sinks: int = 1,
    recent: int = 1,
    softcap: float = 0.0,
    scale: float | None = None,
    return_blocks: bool = False,
    validate: bool = True,
    out: torch.Tensor | None = None,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Batched single-token decode q [B, Hq, D] -> [B, Hq, D] over `budget` blocks of each
    request, chosen for each KV head: the first `sinks` blocks, the last `recent` (at
    least 1: the block being filled needs no bounds), and of the others those with the
    largest score, the largest over the head's queries of

        sum_d max(q_d * min_d, q_d * max_d)

    (of -q where scale is negative), in 64 bits; ties go to the lower block, and a sum that
    is NaN does not count. A request of at most `budget` blocks is read whole.

    With return_blocks also the chosen blocks' places in their request, ascending: int64
    [B, Hkv, budget], -1 past the end. With validate=False a seq_lens of 0 (a padded
    row) gives zeros.
    """
    what = "paged_attention_decode_sparse"
    device, _ = _check(q, k_cache, v_cache, block_size, softcap, None, what)
    _check_bounds(key_bounds, k_cache)
    if key_bounds.device != device:
        raise RuntimeError(f"{what}: operands are on different devices")
    if sinks < 0 or recent < 1 or budget < sinks + recent:
        raise ValueError("budget must be at least sinks + recent, with recent at least 1")
    if budget >= 1 << 31:
        raise ValueError("budget must be below 2^31")
    batch, num_q_heads, head_dim = q.shape
    block_tables = _table(block_tables, batch, device)
    seq_lens = _as_index_tensor(seq_lens, device).contiguous()
    if seq_lens.shape != (batch,):
        raise ValueError("seq_lens length must match batch size of q")
    out = _out(q, out, device)
    num_blocks, _, num_kv_heads, _ = k_cache.shape
    blocks = None
    if return_blocks:
        blocks = torch.empty(batch, num_kv_heads, budget, dtype=torch.long, device=device)
    if batch > 0:
        if validate:
            _validate_tables(block_tables, seq_lens, block_size, num_blocks)
        q = _aligned_q(q)
        width = block_tables.shape[1]
        dcode = _lib.DTYPE_CODES[q.dtype]
        lib = _lib.load()
        with _lib.on(device):
            nbytes = lib.mlr_paged_decode_sparse_workspace_size(
                batch, num_q_heads, num_kv_heads, head_dim, width, block_size, budget, dcode)
            ws = _workspace(nbytes, device)
            status = lib.mlr_paged_decode_sparse(
                q.data_ptr(), q.stride(0), q.stride(1), k_cache.data_ptr(), v_cache.data_ptr(),
                key_bounds.data_ptr(), num_blocks, block_size, num_kv_heads, head_dim,
                block_tables.data_ptr(), block_tables.stride(0), width, seq_lens.data_ptr(),
                batch, num_q_heads, budget, sinks, recent,
                head_dim ** -0.5 if scale is None else scale, softcap,
                dcode, None if blocks is None else blocks.data_ptr(),
                None if ws is None else ws.data_ptr(), nbytes, out.data_ptr(), out.stride(0),
                out.stride(1), _lib.stream_handle(device))
        _lib.check(status, "mlr_paged_decode_sparse")
    return (out, blocks) if return_blocks else out
