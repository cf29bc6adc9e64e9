"""Adaptive draft depth for self-speculative decoding
(moe_prefetch/speculative.py:39-77 `AdaptiveSpeculationPolicy`).

The policy decides, before each decode round, whether to run a plain
single-token step (to calibrate, or because speculation was switched off) or a
draft round of `depth` tokens, whose verify pass is the 1 + depth row batch
this library runs on the batch path (`ExpertParallelStack` with
`batch = 1 + depth`; `bench.py --workload verify` measures 1 + 4):

* calibrate on three plain steps (their step times);
* afterwards compare the median cost per emitted token of the last three
  draft rounds with the median of the three plain steps; when drafting is more
  than 5% slower, halve the depth (its draft history restarts), and at depth 1
  stop drafting for good;
* recalibrate (forget both histories) after 16 draft rounds or 256 tokens of
  context growth since the last plain step.

Depth starts at the requested maximum, clamped to [1, 16].

`verify_rows` is the end of such a round: the verify rows' logits by an 8-bit LM head,
what they say of the drafted tokens, and how many of those are accepted
(speculative.py:121-193 compares greedy choices).
"""
from __future__ import annotations

from typing import List, NamedTuple, Union

CALIBRATE = "calibrate"
PLAIN = "plain"


def _median3(v: List[float]) -> float:
    return sorted(v)[1]


class AdaptiveSpeculationPolicy:
    CALIBRATE, PLAIN = CALIBRATE, PLAIN

    def __init__(self, maximum_depth: int):
        self.depth = max(1, min(16, int(maximum_depth)))
        self.plain: List[float] = []     # the last (up to) three plain step times
        self.draft: List[float] = []     # the last (up to) three draft-round costs per emitted token
        self.stopped = False
        self.baseline_ctx = 0            # context length at the last plain step
        self.rounds_since = 0            # draft rounds since the last recalibration

    def action(self, ctx: int) -> Union[str, int]:
        """PLAIN, CALIBRATE, or the draft depth for a round at context length `ctx`."""
        if self.stopped:
            return PLAIN
        calibrated = len(self.plain) == 3
        if calibrated and (self.rounds_since >= 16 or ctx - self.baseline_ctx >= 256):
            self.plain, self.draft, self.rounds_since = [], [], 0
            calibrated = False
        return self.depth if calibrated else CALIBRATE

    def observe_plain(self, seconds: float, ctx: int) -> None:
        self.plain = (self.plain + [seconds])[-3:]
        self.baseline_ctx = ctx

    def observe_draft(self, seconds: float, emitted: int) -> None:
        """A draft round took `seconds` and emitted `emitted` tokens (>= 1)."""
        self.rounds_since += 1
        self.draft = (self.draft + [seconds / emitted])[-3:]
        if len(self.draft) < 3 or len(self.plain) < 3:
            return
        if _median3(self.draft) > _median3(self.plain) * 1.05:
            if self.depth == 1:
                self.stopped = True
            else:
                self.depth = max(1, self.depth // 2)
                self.draft = []


class VerifyAnswer(NamedTuple):
    """Of a draft of d tokens, on the device: `accepted` () int64, how many are accepted;
    `next_token` () int32, the greedy choice after the last accepted one; `answers`
    (logprobs.TokenLogprobs), per row what it says of its drafted token (the last row has
    none) and its likeliest tokens."""
    accepted: "torch.Tensor"
    next_token: "torch.Tensor"
    answers: "logprobs.TokenLogprobs"


def verify_rows(rows, head, draft, n_top: int = 1) -> VerifyAnswer:
    """The answer of a verify pass. rows: (1 + d, H), the final normalised hidden rows of the
    last token and the d drafted ones; head: the LM head as an `int8.Int8Matrix` (V, H);
    draft: (d,) int32. Row i answers for draft[i]: a drafted token is accepted while every
    one up to it is its row's greedy choice (the largest logit, equal ones by the lower
    id). Nothing is copied to the host."""
    import torch

    from .int8 import int8_linear
    from .logprobs import token_logprobs
    if draft.dim() != 1 or rows.dim() != 2 or rows.shape[0] != draft.shape[0] + 1:
        raise ValueError("rows must be (1 + d, H) for a draft of d tokens")
    if n_top < 1:
        raise ValueError("n_top must be at least 1: the next token is the first of them")
    tokens = torch.cat((draft, draft.new_full((1,), -1)))
    answers = token_logprobs(int8_linear(rows, head, out_dtype=torch.float32), tokens, n_top=n_top)
    accepted = torch.cumprod(answers.rank[:-1] == 0, 0).sum()
    return VerifyAnswer(accepted, answers.top_ids[:, 0].gather(0, accepted.view(1))[0], answers)
