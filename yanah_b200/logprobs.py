"""What rows of logits say of given tokens: log probability and rank, the rows'
entropies and their likeliest alternatives (``yn_token_logprobs``).

``speculation.verify_rows`` accepts a draft with it; it serves as well for scoring
text and for log-probability requests. No counterpart in the reference, which
compares greedy choices (speculative.py:121-193).
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib
from .launch import DTYPES, check_floats, check_like, elsewhere, raw_stream, row_stride, rows_of, run_there


class TokenLogprobs(NamedTuple):
    """Per row: ``logprob`` (T) fp32 and ``rank`` (T) int32 of the given token (0: the
    greedy choice; None without tokens), ``entropy`` (T) fp32 in nats, ``top_ids``
    (T, n) int32 and ``top_logprobs`` (T, n) fp32 of the likeliest tokens (None with
    n_top = 0)."""
    logprob: Optional[torch.Tensor]
    rank: Optional[torch.Tensor]
    entropy: torch.Tensor
    top_ids: Optional[torch.Tensor]
    top_logprobs: Optional[torch.Tensor]


def token_logprobs(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None, n_top: int = 0,
                   stream: Optional[torch.cuda.Stream] = None) -> TokenLogprobs:
    """Rows of logits (T, V) in fp32, bf16 or fp16 and a token (T) int32 of each.

    Tokens that come first have the larger logit, equal ones the lower id; ``rank``
    counts how many come before the given one. Logits of -inf (tokens barred from
    sampling) have no mass and are not listed (id -1, log probability -inf). A row
    of -inf alone has log probabilities of -inf and entropy 0, one with a NaN has NaN
    and ranks and ids of -1. A token outside [0, V), as padded rows have, gives NaN
    and rank -1. n_top <= 64."""
    check_floats(logits, "logits")
    if elsewhere(logits.device, stream):
        return run_there(lambda: token_logprobs(logits, tokens, n_top), logits.device, stream, (logits, tokens))
    logits = rows_of(logits, "logits")
    rows, vocab = logits.shape
    dev = logits.device
    if tokens is not None:
        check_like(tokens, logits, (rows,), (torch.int32,), "tokens")
        tokens = tokens.contiguous()
    if vocab < 1:
        raise ValueError("logits must have at least one column")
    if not 0 <= n_top <= min(64, vocab):
        raise ValueError(f"n_top must be in [0, {min(64, vocab)}], not {n_top}")
    entropy = torch.empty(rows, dtype=torch.float32, device=dev)
    logprob = rank = top_ids = top_lp = None
    if tokens is not None:
        logprob = torch.empty_like(entropy)
        rank = torch.empty_like(tokens)
    if n_top:
        top_ids = torch.empty((rows, n_top), dtype=torch.int32, device=dev)
        top_lp = torch.empty((rows, n_top), dtype=torch.float32, device=dev)
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    _lib.check(_lib.lib().yn_token_logprobs(
        logits.data_ptr(), DTYPES[logits.dtype], row_stride(logits), rows, vocab, ptr(tokens), n_top, ptr(logprob),
        entropy.data_ptr(), ptr(rank), ptr(top_ids), ptr(top_lp), raw_stream(dev)))
    return TokenLogprobs(logprob, rank, entropy, top_ids, top_lp)
