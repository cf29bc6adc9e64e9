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
from .launch import check_floats, check_like, elsewhere, raw_stream, rows_of, run_there


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
    dtype, dev = check_floats(logits, "logits"), logits.get_device()
    if elsewhere(dev, stream):
        return run_there(lambda: token_logprobs(logits, tokens, n_top), logits.device, stream, (logits, tokens))
    logits, rows, vocab, stride = rows_of(logits, "logits")
    if vocab < 1:
        raise ValueError("logits must have at least one column")
    if not 0 <= n_top <= min(64, vocab):
        raise ValueError(f"n_top must be in [0, {min(64, vocab)}], not {n_top}")
    f32, i32, like = torch.float32, torch.int32, torch.empty_like
    entropy = logits.new_empty(rows, dtype=f32)
    logprob = rank = top_ids = top_lp = None
    p_tokens = p_logprob = p_rank = p_ids = p_top = None
    if tokens is not None:
        check_like(tokens, dev, (rows,), (i32,), "tokens")
        tokens = tokens.contiguous()
        logprob, rank = like(entropy), like(entropy, dtype=i32)
        p_tokens, p_logprob, p_rank = tokens.data_ptr(), logprob.data_ptr(), rank.data_ptr()
    if n_top:
        top_ids = logits.new_empty(rows, n_top, dtype=i32)
        top_lp = like(top_ids, dtype=f32)
        p_ids, p_top = top_ids.data_ptr(), top_lp.data_ptr()
    _lib.check(_lib.lib().yn_token_logprobs(logits.data_ptr(), dtype, stride, rows, vocab, p_tokens, n_top, p_logprob,
                                            entropy.data_ptr(), p_rank, p_ids, p_top, raw_stream(dev)))
    return TokenLogprobs(logprob, rank, entropy, top_ids, top_lp)
