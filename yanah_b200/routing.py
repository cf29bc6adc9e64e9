"""Routing of rows of router logits by a rule: softmax or sigmoid scores, a bias for
balance that moves the choice but not the weights, groups of experts, the top k and
their (renormalised) weights.

Beside ``yn_route``, which is the softmax top-k of the reference's models
(mlx_backend.py:308-316). ``PrefillStack(rule=...)`` and ``CudaMoEBackend(rule=...)``
route their layers by such a rule; the ids and weights are those that
``int8.int8_experts`` and the record-based expert kernels take.

    rule = RouteRule(top_k=8, score="sigmoid", n_groups=8, top_groups=4, scale=2.5)
    ids, weights = route_scored(logits, rule, bias=balance)
"""
from __future__ import annotations

import ctypes as C
from functools import lru_cache
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib
from .launch import check_floats, check_like, elsewhere, raw_stream, rows_of, run_there

SCORES = {"softmax": 0, "sigmoid": 1}


class RouteRule(NamedTuple("RouteRule", [("top_k", int), ("score", str), ("n_groups", int), ("top_groups", int),
                                        ("group_top", int), ("norm_topk", bool), ("scale", float)])):
    """How a row chooses its experts.

    top_k: experts per row (<= 31). score: "softmax" or "sigmoid". n_groups: the
    experts in that many equal, consecutive groups, of which a row uses the
    ``top_groups`` best; a group's score is the sum of its ``group_top`` (1 or 2)
    largest choice values. norm_topk: divide the weights by their sum. scale:
    factor of the weights."""
    __slots__ = ()

    def __new__(cls, top_k: int, score: str = "softmax", n_groups: int = 1, top_groups: int = 1, group_top: int = 2,
                norm_topk: bool = True, scale: float = 1.0):
        if score not in SCORES:
            raise ValueError(f"score must be 'softmax' or 'sigmoid', not {score!r}")
        return tuple.__new__(cls, (top_k, score, n_groups, top_groups, group_top, norm_topk, scale))


def check_choice_bias(bias: Optional[torch.Tensor], rule: Optional[RouteRule], layers: int, n_experts: int) -> None:
    """The biases of a stack of layers: a row of fp32 for each of its layers."""
    if bias is None:
        return
    if rule is None:
        raise ValueError("choice_bias needs a rule")
    if tuple(bias.shape) != (layers, n_experts):
        raise ValueError(f"choice_bias must have a row for each layer, ({layers}, {n_experts}), not {tuple(bias.shape)}")
    if bias.dtype is not torch.float32:
        raise TypeError(f"choice_bias must be torch.float32, not {bias.dtype}")


@lru_cache(maxsize=256)
def _rule_struct(rule: RouteRule, n_experts: int) -> _lib.RouteRuleStruct:
    return _lib.RouteRuleStruct(n_experts, rule.top_k, SCORES[rule.score], rule.n_groups, rule.top_groups,
                                rule.group_top, int(rule.norm_topk), rule.scale)


def route_scored(logits: torch.Tensor, rule: RouteRule, bias: Optional[torch.Tensor] = None,
                 available: Optional[torch.Tensor] = None, stream: Optional[torch.cuda.Stream] = None,
                 out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Ids (T, k) int32 and weights (T, k) fp32 of rows of router logits (T, E) in
    fp32, bf16 or fp16.

    The choice value of an expert is its score plus ``bias`` (E) fp32; ids are in
    descending order of it, equal ones by id; the order is that of 64-bit arithmetic.
    The weights are the scores of the chosen. An expert does not take part where
    ``available`` (E) (bool or uint8) is false or its logit is -inf or NaN; rows with
    fewer than k experts left end in ids of -1 with weight 0. Any number of rows.
    ``out``: contiguous ids and weights to write."""
    dtype, dev = check_floats(logits, "logits"), logits.get_device()
    if elsewhere(dev, stream):
        return run_there(lambda: route_scored(logits, rule, bias, available, out=out), logits.device, stream,
                         (logits, bias, available, *(out or ())))
    logits, rows, e, stride = rows_of(logits, "logits")
    if bias is not None:
        check_like(bias, dev, (e,), (torch.float32,), "bias")
        bias = bias.contiguous()
    if available is not None:
        check_like(available, dev, (e,), (torch.bool, torch.uint8), "available")
        available = available.contiguous()
    if out is None:
        ids = logits.new_empty(rows, rule.top_k, dtype=torch.int32)
        weights = torch.empty_like(ids, dtype=torch.float32)
    else:
        ids, weights = out
        check_like(ids, dev, (rows, rule.top_k), (torch.int32,), "out ids")
        check_like(weights, dev, (rows, rule.top_k), (torch.float32,), "out weights")
        if not (ids.is_contiguous() and weights.is_contiguous()):
            raise ValueError("out must be contiguous")
    _lib.check(_lib.lib().yn_route_scored(
        C.byref(_rule_struct(rule, e)), logits.data_ptr(), dtype, stride, rows,
        None if bias is None else bias.data_ptr(), None if available is None else available.data_ptr(),
        ids.data_ptr(), weights.data_ptr(), raw_stream(dev)))
    return ids, weights
