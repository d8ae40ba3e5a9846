"""Log probabilities of given tokens, entropy and the most likely tokens of rows of logits
(csdr_token_logprobs): what a scored text (perplexity) or an answer with alternatives needs beside
the token that select_best_from_logits (api/cortex_sdk.cpp:1005-1030) picks from the same scores.
"""
from __future__ import annotations

import typing

from . import _lib
from .hsdr import _check, _torch
from .paged import _bytes, _dtype, _empty, _int, _on_device, _stream_of


class TokenLogprobs(typing.NamedTuple):
    logprobs: typing.Any      # (rows,) float32, None without tokens
    entropy: typing.Any       # (rows,) float32, nats
    top_ids: typing.Any       # (rows, top_n) int32, likeliest first; None without top_n
    top_logprobs: typing.Any  # (rows, top_n) float32


def token_logprobs(logits, tokens=None, top_n: int = 0, temperature: float = 1.0, workspace=None,
                   stream=None) -> TokenLogprobs:
    """logits: (rows, n) float32 or float16 on the device, rows any stride apart; tokens: (rows,)
    int32, negative for none. A row with a NaN or +infinity has NaN log probabilities, and only its
    finite logits among the top. Without rows nothing is done. With `stream` the call runs and
    allocates there, ordered by the caller."""
    torch = _torch()
    lib, top_n = _lib.load(), _int(top_n)
    dt = _dtype(logits)
    if logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError("logits must be (rows, n) with a row's values side by side")
    rows, n = logits.shape
    if rows > 1 and logits.stride(0) < n:  # an expanded tensor, or rows that overlap
        raise ValueError("the rows of logits overlap")
    if tokens is not None and (tokens.dtype != torch.int32 or tuple(tokens.shape) != (rows,) or
                               not tokens.is_contiguous()):
        raise ValueError("tokens must be a contiguous int32 tensor, one per row")
    index = _on_device(torch, "tensors", logits, tokens, workspace)
    dev = logits.device
    if workspace is None and rows > 0:
        need = lib.csdr_token_logprobs_workspace_bytes(rows, n, top_n)
        workspace = _empty(torch, need, torch.uint8, dev, stream) if need else None
    lp, entropy = _empty(torch, (2, rows), torch.float32, dev, stream).unbind(0)
    ids = top = None
    if 0 < top_n <= 64:  # (else the library refuses it)
        ids = _empty(torch, (rows, top_n), torch.int32, dev, stream)
        top = _empty(torch, (rows, top_n), torch.float32, dev, stream)
    if tokens is None:
        lp = None
    if rows == 0:
        return TokenLogprobs(lp, entropy, ids, top)
    _check(lib.csdr_token_logprobs(
        logits.data_ptr(), dt, rows, n, logits.stride(0) if rows > 1 else 0, temperature,
        tokens.data_ptr() if tokens is not None else None,
        lp.data_ptr() if lp is not None else None, entropy.data_ptr(), top_n,
        ids.data_ptr() if ids is not None else None, top.data_ptr() if top is not None else None,
        workspace.data_ptr() if workspace is not None else None,
        _bytes(workspace) if workspace is not None else 0, _stream_of(torch, index, stream)))
    return TokenLogprobs(lp, entropy, ids, top)
