"""Paged attention with capped or biased scores, with prefixes that are seen
whole, and over a prefix that a decode batch shares (csrc/scored_rows.hip,
csrc/scored_tiles.hip, csrc/scored_attention.hip). No reference counterpart; beside the plain calls of
``paged_attention``, with the same caches, tables and packed batches.

For the query at position i of head h and a key at j:

    x = scale * q.k
    softcap > 0:   x = softcap * tanh(x / softcap)
    alibi_slopes:  x = x - alibi_slopes[h] * |i - j|

and the result is the softmax of x over the visible keys, times V. bf16, fp16
and FP32; head_dim a multiple of 8 (FP32: 4) up to 128; any block size. Scores,
statistics and sums are FP32, whatever the type. In bf16 and fp16 the probabilities
are rounded to the type before they meet V, at every head size, and a capped score is
within 9e-7 of its own size.

Workspaces come from torch's allocator on the current stream, call by call, so
calls on different streams, or captured into different graphs, never share one.
"""

from __future__ import annotations

import torch

from .. import _lib
from .paged_attention import (_as_index_tensor, _check_cache_pair, _raise_table_errors,
                              _require_kernel_layout, _validate_tables)


def _check(q, k_cache, v_cache, block_size, softcap, alibi_slopes, what):
    if q.ndim != 3:
        raise ValueError("q must have shape [num_tokens, Hq, D]")
    _check_cache_pair(k_cache, v_cache)
    num_q_heads, head_dim = q.shape[1], q.shape[2]
    num_kv_heads = k_cache.shape[2]
    if head_dim != k_cache.shape[3]:
        raise ValueError("q and KV cache must have the same head_dim")
    if num_q_heads == 0 or num_kv_heads == 0 or num_q_heads % num_kv_heads != 0:
        raise ValueError("num_query_heads must be divisible by num_kv_heads")
    if block_size != k_cache.shape[1]:
        raise ValueError("block_size does not match KV cache layout")
    step = 4 if q.dtype == torch.float32 else 8
    if q.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise TypeError(f"{what}: unsupported dtype {q.dtype}")
    if head_dim % step or not 0 < head_dim <= 128:
        raise ValueError(f"{what} takes head_dim in multiples of {step} up to 128")
    if softcap != 0 and not 1e-30 <= softcap <= 1e30:
        raise ValueError("softcap must be 0 (off) or a positive number in [1e-30, 1e30]")
    _require_kernel_layout(q, k_cache, v_cache, what)
    if alibi_slopes is not None:
        if alibi_slopes.shape != (num_q_heads,) or alibi_slopes.dtype != torch.float32:
            raise ValueError("alibi_slopes must be an FP32 tensor of shape [Hq]")
        alibi_slopes = alibi_slopes.contiguous()
        return _lib.require_hip(q, k_cache, v_cache, alibi_slopes, what=what), alibi_slopes
    return _lib.require_hip(q, k_cache, v_cache, what=what), None


def _aligned_q(q: torch.Tensor) -> torch.Tensor:
    """q with unit stride and rows at multiples of 16 bytes."""
    step = 16 // q.element_size()
    if (q.stride(2) != 1 or q.stride(0) % step or q.stride(1) % step or q.data_ptr() % 16):
        q = q.clone(memory_format=torch.contiguous_format)
    return q


def _out(q: torch.Tensor, out: torch.Tensor | None, device) -> torch.Tensor:
    if out is None:
        return torch.empty(q.shape, dtype=q.dtype, device=device)
    if out.shape != q.shape or out.dtype != q.dtype or out.device != device or (
            out.numel() and out.stride(2) != 1):
        raise ValueError("out must match q in shape, dtype and device, with contiguous rows")
    return out


def _table(block_tables, rows: int, device: torch.device) -> torch.Tensor:
    block_tables = _as_index_tensor(block_tables, device)
    if block_tables.ndim != 2 or block_tables.shape[0] != rows:
        raise ValueError("block_tables must have shape [num_sequences, max_num_blocks]")
    return block_tables if block_tables.stride(1) == 1 else block_tables.contiguous()


def _workspace(nbytes: int, device: torch.device) -> torch.Tensor | None:
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def paged_attention_decode_scored(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_tables: torch.Tensor,
    seq_lens: torch.Tensor,
    block_size: int,
    *,
    softcap: float = 0.0,
    alibi_slopes: torch.Tensor | None = None,
    scale: float | None = None,
    validate: bool = True,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Batched single-token decode: q [B, Hq, D] -> [B, Hq, D], the query of
    request b at position seq_lens[b] - 1 over keys [0, seq_lens[b]).

    Operands and checks as for paged_attention_decode_batch_parallel. With
    validate=False, for callers that check a step's metadata once, a seq_lens of 0
    (a padded row) gives zeros.
    """
    what = "paged_attention_decode_scored"
    device, slopes = _check(q, k_cache, v_cache, block_size, softcap, alibi_slopes, what)
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
    q = _aligned_q(q)
    width = block_tables.shape[1]
    lib = _lib.load()
    with _lib.on(device):
        nbytes = lib.mlr_paged_decode_scored_workspace_size(
            batch, num_q_heads, num_kv_heads, head_dim, width * block_size)
        ws = _workspace(nbytes, device)
        status = lib.mlr_paged_decode_scored(
            q.data_ptr(), q.stride(0), q.stride(1), k_cache.data_ptr(), v_cache.data_ptr(),
            num_blocks, block_size, num_kv_heads, head_dim, block_tables.data_ptr(),
            block_tables.stride(0), width, seq_lens.data_ptr(), batch, num_q_heads,
            head_dim ** -0.5 if scale is None else scale, softcap,
            None if slopes is None else slopes.data_ptr(), _lib.DTYPE_CODES[q.dtype],
            None if ws is None else ws.data_ptr(), nbytes, out.data_ptr(), out.stride(0),
            out.stride(1), _lib.stream_handle(device))
    _lib.check(status, "mlr_paged_decode_scored")
    return out


def _validate_prefill(block_tables, query_start_loc, context_lens, prefix_lens, block_size,
                      num_blocks, total_q, max_query_len=None) -> None:
    """One host sync for all metadata checks of a packed batch."""
    width = block_tables.shape[1]
    lens = query_start_loc[1:] - query_start_loc[:-1]
    required = torch.div(context_lens + (block_size - 1), block_size, rounding_mode="floor")
    used = torch.arange(width, device=block_tables.device)[None, :] < required[:, None]
    bad = used & ((block_tables < 0) | (block_tables >= num_blocks))
    flags = [query_start_loc[0] != 0, (lens < 0).any(), query_start_loc[-1] != total_q,
             (context_lens < lens).any(), (required > width).any(), bad.any()]
    flags.append((lens > (total_q if max_query_len is None else max_query_len)).any())
    if prefix_lens is not None:
        flags.append(((prefix_lens < 0) | (prefix_lens > context_lens)).any())
    flags = torch.stack(flags).tolist()
    if flags[0]:
        raise ValueError("query_start_loc must start at 0")
    if flags[1]:
        raise ValueError("query_start_loc must not decrease")
    if flags[2]:
        raise ValueError("query_start_loc must end at the packed token count")
    if flags[3]:
        raise ValueError("context_lens must cover each request's tokens")
    _raise_table_errors(False, flags[4], flags[5])
    if flags[6]:
        raise ValueError("max_query_len must cover the longest chunk")
    if prefix_lens is not None and flags[7]:
        raise ValueError("prefix_lens must lie between 0 and context_lens")


def paged_attention_prefill_scored(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_tables: torch.Tensor,
    query_start_loc: torch.Tensor,
    context_lens: torch.Tensor,
    block_size: int,
    *,
    softcap: float = 0.0,
    alibi_slopes: torch.Tensor | None = None,
    prefix_lens: torch.Tensor | None = None,
    scale: float | None = None,
    max_query_len: int | None = None,
    validate: bool = True,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Chunk prefill of a packed batch (ModelBatch layout): q [total_q, Hq, D],
    sequence s's rows at [query_start_loc[s], query_start_loc[s+1]), the last of
    its context_lens[s] positions, whose keys are all in the cache.

    The query at position i sees the keys j <= i, and with prefix_lens [S] also
    all j < prefix_lens[s], those ahead of it included (a prompt whose first part
    attends to itself in both directions). Rows past query_start_loc[-1] are not
    written. max_query_len, at least the longest chunk, saves a host sync;
    validate=False skips the metadata checks, for callers that make them once a step.
    """
    what = "paged_attention_prefill_scored"
    device, slopes = _check(q, k_cache, v_cache, block_size, softcap, alibi_slopes, what)
    total_q, num_q_heads, head_dim = q.shape
    query_start_loc = _as_index_tensor(query_start_loc, device).contiguous()
    if query_start_loc.ndim != 1 or query_start_loc.shape[0] == 0:
        raise ValueError("query_start_loc must have shape [num_sequences + 1]")
    seqs = query_start_loc.shape[0] - 1
    block_tables = _table(block_tables, seqs, device)
    context_lens = _as_index_tensor(context_lens, device).contiguous()
    if context_lens.shape != (seqs,):
        raise ValueError("context_lens must hold one length per sequence")
    if prefix_lens is not None:
        prefix_lens = _as_index_tensor(prefix_lens, device).contiguous()
        if prefix_lens.shape != (seqs,):
            raise ValueError("prefix_lens must hold one length per sequence")
    out = _out(q, out, device)
    num_blocks, _, num_kv_heads, _ = k_cache.shape
    if validate:
        _validate_prefill(block_tables, query_start_loc, context_lens, prefix_lens, block_size,
                          num_blocks, total_q, max_query_len)
    if seqs == 0 or total_q == 0:
        return out
    if max_query_len is None:
        max_query_len = int((query_start_loc[1:] - query_start_loc[:-1]).max().item())
    elif max_query_len < 0:
        raise ValueError("max_query_len cannot be negative")
    max_query_len = min(max_query_len, total_q)
    q = _aligned_q(q)
    width = block_tables.shape[1]
    dcode = _lib.DTYPE_CODES[q.dtype]
    lib = _lib.load()
    with _lib.on(device):
        nbytes = lib.mlr_paged_prefill_scored_workspace_size(
            seqs, max_query_len, width, block_size, num_q_heads, num_kv_heads, head_dim, dcode)
        ws = _workspace(nbytes, device)
        status = lib.mlr_paged_prefill_scored(
            q.data_ptr(), q.stride(0), q.stride(1), k_cache.data_ptr(), v_cache.data_ptr(),
            num_blocks, block_size, num_kv_heads, head_dim, block_tables.data_ptr(),
            block_tables.stride(0), width, query_start_loc.data_ptr(), context_lens.data_ptr(),
            None if prefix_lens is None else prefix_lens.data_ptr(), seqs, total_q, max_query_len,
            num_q_heads, head_dim ** -0.5 if scale is None else scale, softcap,
            None if slopes is None else slopes.data_ptr(), dcode,
            None if ws is None else ws.data_ptr(), nbytes, out.data_ptr(), out.stride(0),
            out.stride(1), _lib.stream_handle(device))
    _lib.check(status, "mlr_paged_prefill_scored")
    return out


def paged_attention_decode_shared_prefix(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    prefix_table: torch.Tensor,
    prefix_len: int,
    block_tables: torch.Tensor,
    seq_lens: torch.Tensor,
    block_size: int,
    *,
    softcap: float = 0.0,
    alibi_slopes: torch.Tensor | None = None,
    scale: float | None = None,
    validate: bool = True,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """paged_attention_decode_scored for a batch whose requests share their
    first prefix_len positions: these are read once for all requests, through
    prefix_table [num_blocks of the prefix]; positions from prefix_len on through
    block_tables [B, W], which are indexed by position as ever (entries before
    prefix_len // block_size are not read, so tables that repeat the prefix's blocks
    serve as they are). seq_lens [B] count the prefix; the prefix may end inside
    a block, whose rest is then each request's own.

    With validate=False a request with seq_lens[b] < prefix_len sees its first
    seq_lens[b] positions, and none, with a result of zeros, if that is 0.
    """
    what = "paged_attention_decode_shared_prefix"
    device, slopes = _check(q, k_cache, v_cache, block_size, softcap, alibi_slopes, what)
    batch, num_q_heads, head_dim = q.shape
    prefix_table = _as_index_tensor(prefix_table, device).contiguous()
    if prefix_table.ndim != 1:
        raise ValueError("prefix_table must have shape [num_blocks]")
    if prefix_len < 0:
        raise ValueError("prefix_len cannot be negative")
    needed = -(-prefix_len // block_size)
    if prefix_table.shape[0] < needed:
        raise ValueError("prefix_table does not contain enough blocks for prefix_len")
    block_tables = _table(block_tables, batch, device)
    seq_lens = _as_index_tensor(seq_lens, device).contiguous()
    if seq_lens.shape != (batch,):
        raise ValueError("seq_lens length must match batch size of q")
    out = _out(q, out, device)
    if batch == 0:
        return out
    num_blocks, _, num_kv_heads, _ = k_cache.shape
    width = block_tables.shape[1]
    if validate:
        first = prefix_len // block_size
        required = torch.div(seq_lens + (block_size - 1), block_size, rounding_mode="floor")
        # A request that ends with the prefix needs no block of its own.
        required = torch.where(seq_lens > prefix_len, required, 0)
        column = torch.arange(width, device=device)[None, :]
        used = (column >= first) & (column < required[:, None])
        prefix = prefix_table[:needed]
        flags = torch.stack([
            (seq_lens <= 0).any(), (required > width).any(),
            (used & ((block_tables < 0) | (block_tables >= num_blocks))).any(),
            (seq_lens < prefix_len).any(),
            ((prefix < 0) | (prefix >= num_blocks)).any()]).tolist()
        _raise_table_errors(*flags[:3])
        if flags[3]:
            raise ValueError("seq_lens must be at least prefix_len")
        if flags[4]:
            raise ValueError("prefix_table contains an invalid physical block")
    q = _aligned_q(q)
    dcode = _lib.DTYPE_CODES[q.dtype]
    lib = _lib.load()
    with _lib.on(device):
        nbytes = lib.mlr_paged_decode_shared_prefix_workspace_size(
            batch, num_q_heads, num_kv_heads, head_dim, prefix_len, width, block_size, dcode)
        ws = _workspace(nbytes, device)
        status = lib.mlr_paged_decode_shared_prefix(
            q.data_ptr(), q.stride(0), q.stride(1), k_cache.data_ptr(), v_cache.data_ptr(),
            num_blocks, block_size, num_kv_heads, head_dim, prefix_table.data_ptr(),
            prefix_table.shape[0], prefix_len, block_tables.data_ptr(), block_tables.stride(0),
            width, seq_lens.data_ptr(), batch, num_q_heads,
            head_dim ** -0.5 if scale is None else scale, softcap,
            None if slopes is None else slopes.data_ptr(), dcode,
            None if ws is None else ws.data_ptr(), nbytes, out.data_ptr(), out.stride(0),
            out.stride(1), _lib.stream_handle(device))
    _lib.check(status, "mlr_paged_decode_shared_prefix")
    return out
