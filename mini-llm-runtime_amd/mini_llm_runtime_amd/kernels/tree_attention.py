"""Attention for trees of drafted tokens over the paged cache (csrc/tree_attention.hip,
csrc/scored_rows.hip, csrc/scored_tiles.hip). No reference counterpart; beside the packed
prefill of ``scored_attention``, with the same caches, tables and packed batches.

A step that verifies drafted tokens appends the keys and values of all of them to the
cache, in any order in which the batch's rows have them, and asks for each one's
attention over the keys before the drafted ones and over its own ancestors. Which
these are is a row of bits a token, made once a step from the tokens' parents
(``tree_ancestors``) or by the caller. ``key_eviction.compact_keys`` then moves the
accepted path's rows together.

bf16, fp16 and FP32; head_dim a multiple of 8 (FP32: 4) up to 128; any block size.
Scores, statistics and sums are FP32, whatever the type, a probability meets V to 2^-15 of
itself in bf16 and 2^-21 in fp16, and the result is rounded once.
"""

from __future__ import annotations

import torch

from .. import _lib
from .paged_attention import _as_index_tensor
from .scored_attention import _aligned_q, _check, _out, _table, _validate_prefill, _workspace


def tree_ancestors(
    parents: torch.Tensor,
    query_start_loc: torch.Tensor,
    max_nodes: int,
    *,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Each drafted token's ancestors, and itself, as bits: int64
    [total_q, ceil(max_nodes / 64)], bit j % 64 of word j // 64 for token j of the
    same sequence.

    parents [total_q] holds each token's parent as a place in its own sequence, whose
    rows are [query_start_loc[s], query_start_loc[s+1]); a place out of range (-1) is
    none. Parents may stand behind their children. max_nodes, up to 4096, is at least the
    longest sequence: tokens past it have no bit, and those past 4096 no row.
    """
    what = "tree_ancestors"
    if parents.ndim != 1:
        raise ValueError("parents must have shape [total_q]")
    if not 0 < max_nodes <= 4096:
        raise ValueError("max_nodes must be greater than 0 and at most 4096")
    device = _lib.require_hip(parents, what=what)
    parents = _as_index_tensor(parents, device).contiguous()
    query_start_loc = _as_index_tensor(query_start_loc, device).contiguous()
    if query_start_loc.ndim != 1 or query_start_loc.shape[0] == 0:
        raise ValueError("query_start_loc must have shape [num_sequences + 1]")
    shape = (parents.shape[0], (max_nodes + 63) // 64)
    if out is None:
        out = torch.zeros(shape, dtype=torch.long, device=device)
    elif (out.shape != shape or out.dtype != torch.long or out.device != device
          or not out.is_contiguous()):
        raise ValueError("out must be a contiguous int64 tensor [total_q, ceil(max_nodes / 64)]")
    with _lib.on(device):
        status = _lib.load().mlr_tree_ancestors(
            parents.data_ptr(), query_start_loc.data_ptr(), query_start_loc.shape[0] - 1,
            shape[0], shape[1], out.data_ptr(), _lib.stream_handle(device))
    _lib.check(status, "mlr_tree_ancestors")
    return out


def _validate_words(query_start_loc, words) -> None:
    """For a max_query_len that the words may not cover: whether they cover the sequences."""
    if ((query_start_loc[1:] - query_start_loc[:-1]) > 64 * words).any():
        raise ValueError("ancestors must hold a bit for every drafted token of a sequence")


def paged_attention_tree(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_tables: torch.Tensor,
    query_start_loc: torch.Tensor,
    context_lens: torch.Tensor,
    ancestors: torch.Tensor,
    block_size: int,
    *,
    softcap: float = 0.0,
    scale: float | None = None,
    max_query_len: int | None = None,
    validate: bool = True,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Packed drafted tokens q [total_q, Hq, D], sequence s's at the rows
    [query_start_loc[s], query_start_loc[s+1]), whose keys are the last of the
    context_lens[s] in the cache, in the same order.

    A row sees every key before the drafted ones, and drafted token j of its sequence if
    bit j % 64 of ancestors[row, j // 64] is set: int64 [total_q, words], any bits, not
    only those of a tree. A row that sees no key gets zeros. Rows past
    query_start_loc[-1] are not written. max_query_len, at least the most tokens of a
    sequence, saves a host sync; validate=False skips the checks of the metadata's
    values, for callers that make them once a step.
    """
    what = "paged_attention_tree"
    device, _ = _check(q, k_cache, v_cache, block_size, softcap, None, what)
    total_q, num_q_heads, head_dim = q.shape
    query_start_loc = _as_index_tensor(query_start_loc, device).contiguous()
    if query_start_loc.ndim != 1 or query_start_loc.shape[0] == 0:
        raise ValueError("query_start_loc must have shape [num_sequences + 1]")
    seqs = query_start_loc.shape[0] - 1
    block_tables = _table(block_tables, seqs, device)
    context_lens = _as_index_tensor(context_lens, device).contiguous()
    if context_lens.shape != (seqs,):
        raise ValueError("context_lens must hold one length per sequence")
    if ancestors.ndim != 2 or ancestors.shape[0] != total_q or ancestors.shape[1] == 0:
        raise ValueError("ancestors must have shape [total_q, words]")
    if ancestors.dtype != torch.long or ancestors.device != device:
        raise ValueError("ancestors must be an int64 tensor on the device of q")
    ancestors = ancestors.contiguous()
    words = ancestors.shape[1]
    out = _out(q, out, device)
    num_blocks, _, num_kv_heads, _ = k_cache.shape
    if validate:
        _validate_prefill(block_tables, query_start_loc, context_lens, None, block_size,
                          num_blocks, total_q, max_query_len)
    if seqs == 0 or total_q == 0:
        return out
    if max_query_len is None:
        max_query_len = int((query_start_loc[1:] - query_start_loc[:-1]).max().item())
    elif max_query_len < 0:
        raise ValueError("max_query_len cannot be negative")
    max_query_len = min(max_query_len, total_q)
    if validate and max_query_len > 64 * words:
        _validate_words(query_start_loc, words)
    q = _aligned_q(q)
    width = block_tables.shape[1]
    dcode = _lib.DTYPE_CODES[q.dtype]
    lib = _lib.load()
    with _lib.on(device):
        nbytes = lib.mlr_paged_attention_tree_workspace_size(
            seqs, max_query_len, width, block_size, num_q_heads, num_kv_heads, head_dim, dcode)
        ws = _workspace(nbytes, device)
        status = lib.mlr_paged_attention_tree(
            q.data_ptr(), q.stride(0), q.stride(1), k_cache.data_ptr(), v_cache.data_ptr(),
            num_blocks, block_size, num_kv_heads, head_dim, block_tables.data_ptr(),
            block_tables.stride(0), width, query_start_loc.data_ptr(), context_lens.data_ptr(),
            ancestors.data_ptr(), words, seqs, total_q, max_query_len, num_q_heads,
            head_dim ** -0.5 if scale is None else scale, softcap, dcode,
            None if ws is None else ws.data_ptr(), nbytes, out.data_ptr(), out.stride(0),
            out.stride(1), _lib.stream_handle(device))
    _lib.check(status, "mlr_paged_attention_tree")
    return out
