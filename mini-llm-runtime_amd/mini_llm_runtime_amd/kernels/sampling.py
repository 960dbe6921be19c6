"""Sampling with temperature, top-k, top-p and min-p on the HIP library
(csrc/sampling.hip): one given random number a row, the same token for the same
logits and numbers always; one launch, or four over a few long rows. No reference counterpart: the
reference decodes greedily (runtime/model_runner.py:287-322)."""

from __future__ import annotations

import torch

from .. import _lib

_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def sample_tokens(logits: torch.Tensor, uniforms: torch.Tensor, *,
                  temperature: float | torch.Tensor = 1.0, top_k: int | torch.Tensor = 0,
                  top_p: float | torch.Tensor = 1.0, min_p: float | torch.Tensor = 0.0,
                  rows: torch.Tensor | None = None, return_logprobs: bool = False):
    """One token id per row: logits [N, vocab] (bf16, fp16 or FP32, unit stride
    along the vocabulary) and uniforms [B] in [0, 1) (FP32 or FP64) -> int64 [B],
    and with return_logprobs also FP32 [B], the log-probability under what was
    kept. Row b reads logits row rows[b] (int64 [B]), or b where rows is None.

    temperature, top_k, top_p and min_p are numbers or tensors [B] (FP32; top_k
    int32 or int64). With w_i = exp((x_i - max x) / temperature) and the tokens in
    descending order of their logits, equal ones by index, kept are: the first
    top_k (all if top_k <= 0); of those the shortest head that weighs at least
    top_p times their sum (all if top_p >= 1, one if top_p <= 0); of those the ones
    with w_i >= min_p, the first always. The token is the first of the order whose
    running sum exceeds uniforms[b] times the sum of the kept.

    A temperature of 0 or an infinite largest logit gives the first of the order
    (logprob 0); a row without a logit above -inf, or a rows[b] out of range, -1
    (-inf). Logits of -inf or NaN are never drawn. Weights are held to 2^-44 of the
    largest (less finely past 2^18 tokens), so a token of less than half of that is
    not drawn either.
    """
    if logits.ndim != 2 or logits.shape[1] == 0:
        raise ValueError("logits must have shape [num_rows, vocab]")
    if logits.dtype not in _DTYPES:
        raise TypeError(f"logits dtype {logits.dtype} is not supported")
    total, vocab = logits.shape
    if vocab > 1 << 23:
        raise ValueError("sample_tokens takes vocabularies of up to 2^23 tokens")
    if uniforms.ndim != 1 or uniforms.dtype not in (torch.float32, torch.float64):
        raise ValueError("uniforms must be an FP32 or FP64 tensor of shape [num_rows]")
    count = uniforms.shape[0]
    operands = [logits, uniforms]
    if rows is None:
        if total != count:
            raise ValueError("uniforms must hold one number per logits row")
    elif rows.shape != (count,) or rows.dtype != torch.long:
        raise ValueError("rows must be an int64 tensor shaped like uniforms")
    else:
        rows = rows.contiguous()
        operands.append(rows)
    keep = []  # contiguous copies live until the launch is queued
    args = {}
    for name, value in (("temperature", temperature), ("top_k", top_k), ("top_p", top_p),
                        ("min_p", min_p)):
        if not isinstance(value, torch.Tensor):
            args[name] = (None, value)
            continue
        whole = name == "top_k"
        if value.shape != (count,) or (value.dtype not in _lib.INDEX_CODES if whole
                                       else value.dtype != torch.float32):
            raise ValueError(f"{name} must be a number or "
                             f"{'an integer' if whole else 'an FP32'} tensor shaped like uniforms")
        value = value.contiguous()
        keep.append(value)
        args[name] = (value.data_ptr(), 0)
    uniforms = uniforms.contiguous()
    if vocab > 1 and logits.stride(1) != 1:
        raise ValueError("logits must be unit-stride along the vocabulary")
    stride = logits.stride(0) if total > 1 else vocab
    if stride < vocab:
        raise ValueError("logits rows must not overlap")
    device = _lib.require_hip(*operands, *keep, what="sample_tokens")
    tokens = torch.empty(count, dtype=torch.long, device=device)
    logprobs = torch.empty(count, dtype=torch.float32, device=device) if return_logprobs else None
    if count:
        index = _lib.INDEX_CODES[top_k.dtype] if args["top_k"][0] is not None else 1
        lib = _lib.load()
        with _lib.on(device):
            nbytes = lib.mlr_sample_tokens_workspace_size(count, vocab)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
            status = lib.mlr_sample_tokens(
                logits.data_ptr(), stride, total, _lib.DTYPE_CODES[logits.dtype],
                None if rows is None else rows.data_ptr(), uniforms.data_ptr(),
                uniforms.dtype == torch.float64, *args["temperature"], args["top_k"][0], index,
                args["top_k"][1], *args["top_p"], *args["min_p"], tokens.data_ptr(),
                None if logprobs is None else logprobs.data_ptr(), count, vocab,
                None if ws is None else ws.data_ptr(), nbytes, _lib.stream_handle(device))
        _lib.check(status, "mlr_sample_tokens")
    return (tokens, logprobs) if return_logprobs else tokens
