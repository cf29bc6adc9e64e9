"""GPU tests of the scored router against a plain 64-bit implementation.

Ids are compared for equality: the operator orders as exact arithmetic does. The
weights are fp32: three roundings of 2^-24 (division, scale, sum of at most 31) and
expf within 2 ulp give less than 40 * 2^-24 = 2.4e-6 of a weight; 4e-6 is asked.
"""
from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from tests import ref64
from yanah_b200 import _lib
from yanah_b200.routing import RouteRule, route_scored

pytestmark = pytest.mark.gpu
TOL = 4e-6


def check(z, rule, bias=None, available=None):
    ids, w = route_scored(z, rule, bias=bias, available=available)
    torch.cuda.synchronize()
    ri, rw = ref64.route(z.float().cpu().numpy(), rule.top_k, rule.score, None if bias is None else bias.cpu().numpy(),
                         None if available is None else available.cpu().numpy(), rule.n_groups, rule.top_groups,
                         rule.group_top, rule.norm_topk, rule.scale)
    assert np.array_equal(ids.cpu().numpy(), ri)
    w = w.cpu().numpy()
    assert np.all(np.abs(w - rw) <= TOL * np.abs(rw) + 1e-37)
    return ids, w


def logits(T, E, dtype=torch.float32, seed=0, std=1.5):
    g = torch.Generator().manual_seed(seed)
    return (std * torch.randn(T, E, generator=g)).to(dtype).cuda()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,k,G,kept", [(1, 512, 10, 1, 1), (5, 64, 4, 1, 1), (33, 256, 8, 8, 4), (7, 1024, 31, 1, 1),
                                          (3, 1, 1, 1, 1), (4, 97, 3, 1, 1), (9, 60, 6, 5, 2), (6, 1020, 9, 17, 3),
                                          (2, 1024, 16, 32, 7), (4, 64, 2, 32, 1), (3, 24, 5, 3, 3)])
def test_shapes(dtype, score, T, E, k, G, kept):
    z = logits(T, E, dtype, seed=T * E)
    bias = 0.2 * logits(1, E, seed=9)[0]
    for b in (None, bias):
        for norm, gt in ((True, 2), (False, 1)):
            check(z, RouteRule(k, score, G, kept, gt, norm, 2.5), bias=b)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_masks(score):
    E, k = 64, 4
    z = logits(12, E, seed=3)
    z[0] = -torch.inf                      # nothing left
    z[1, 2:] = -torch.inf                  # fewer than k
    z[2, 5] = torch.nan                    # NaN takes no part
    z[3, 7] = torch.inf
    z[4, 3] = z[4, 40] = torch.inf
    z[5] = torch.finfo(torch.float32).min  # a row at the type's lowest value
    z[6, ::2] = torch.finfo(torch.float32).min
    z[7] = 0.25                            # all equal: the lowest ids
    z[8] = -95.0 - torch.arange(E, device="cuda").float() / 8   # scores below fp32's range
    z[9] = 60.0 + torch.arange(E, device="cuda").float() / 8    # sigmoids that round to one
    away = torch.ones(E, dtype=torch.bool, device="cuda")
    away[::3] = False
    bias = 0.1 * logits(1, E, seed=4)[0]
    for av in (None, away, away.to(torch.uint8), torch.zeros_like(away)):
        for b in (None, bias):
            for G, kept in ((1, 1), (8, 3)):
                check(z, RouteRule(k, score, G, kept), bias=b, available=av)
    bias[3], bias[4] = -torch.inf, torch.nan
    check(z, RouteRule(k, score), bias=bias)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_signed_zeros_are_equal(score):
    z = torch.full((3, 64), -1.0, device="cuda")
    z[:, 5] = -0.0
    z[:, 40] = 0.0
    z[1, 63] = 1e-45
    z[2, 0] = -1e-45
    bias = torch.zeros(64, device="cuda")
    bias[40] = -0.0
    for rule in (RouteRule(4, score), RouteRule(4, score, 8, 3), RouteRule(4, score, 8, 3, 1)):
        check(z, rule)
    # (with a bias the order is that of scores in 64 bits, where 1e-45 is nothing: rows of zeros alone)
    check(z[:1], RouteRule(4, score), bias=bias)
    check(z[:1], RouteRule(4, score, 8, 3), bias=bias)


def test_poisoned_places_do_not_leak():
    # infinities and NaN at experts that are away change nothing
    E = 128
    z = logits(6, E, seed=5)
    av = torch.rand(E, generator=torch.Generator().manual_seed(1)) < 0.5
    av = av.cuda()
    ref = route_scored(z, RouteRule(8), available=av)
    bad = z.clone()
    bad[:, ~av] = torch.nan
    bad[::2, ~av] = torch.inf
    got = route_scored(bad, RouteRule(8), available=av)
    assert all(torch.equal(a, b) for a, b in zip(ref, got))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_near_ties_follow_exact_arithmetic(score):
    # biases that bring choice values within a few fp32 ulp of each other: the order must still be the exact one
    E, T = 64, 400
    z = logits(T, E, seed=11, std=1.0)
    s = torch.softmax(z.double(), 1) if score == "softmax" else torch.sigmoid(z.double())
    # bias that equalises the choice values of row 0 up to rounding, so every row near row 0 is full of near ties
    bias = (1.0 - s[0]).float()
    z = z[0].repeat(T, 1)
    z += 1e-7 * logits(T, E, seed=12)
    check(z, RouteRule(8, score), bias=bias)
    check(z, RouteRule(8, score, 8, 3), bias=bias)
    # equal logits, equal biases: the lowest ids, whatever lies behind the last place
    zero = torch.zeros(E, device="cuda")
    check(torch.ones(3, E, device="cuda"), RouteRule(8, score), bias=zero)
    check(logits(50, E, torch.bfloat16, seed=13).round(), RouteRule(8, score, 4, 2), bias=zero)


@pytest.mark.parametrize("G,kept", [(32, 5), (8, 3)])
def test_group_scores_with_large_biases(G, kept):
    # a group's second value far below its first: its rounding to fp32 (2^-24 of 1000) is larger than the
    # distance of many groups' scores, which the order has to settle all the same
    E, T = 64, 700
    z = logits(T, E, seed=G, std=0.01)
    bias = torch.full((E,), -1000.0, device="cuda")
    bias[::E // G] = 0.25
    check(z, RouteRule(3, "sigmoid", G, kept), bias=bias)
    check(z, RouteRule(3, "softmax", G, kept), bias=bias)


def test_strides_alignment_and_many_rows():
    E = 48
    base = logits(70, 2 * E + 3, torch.bfloat16, seed=6)
    check(base[:, 1:E + 1], RouteRule(5, "sigmoid"))
    check(base[::2, :E], RouteRule(5))
    check(base.t()[:E].t(), RouteRule(5))              # row-strided view
    check(base[:, ::2][:, :E], RouteRule(5))           # elements apart: copied
    check(base[:1].expand(4, -1)[:, :E], RouteRule(5))  # overlapping rows: copied
    z = logits(70000, 16, seed=7)
    ids, w = route_scored(z, RouteRule(2))
    some = torch.tensor([0, 1, 34567, 69999], device="cuda")
    ri, rw = ref64.route(z[some].cpu().numpy(), 2)
    assert np.array_equal(ids[some].cpu().numpy(), ri)
    ids, w = route_scored(z[:0], RouteRule(2))
    assert ids.shape == (0, 2) and w.shape == (0, 2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("E,G", [(64, 1), (128, 4), (256, 8), (512, 16), (1024, 32)])
def test_rows_that_start_anywhere(dtype, E, G):
    # aligned rows of whole lanes are read in wide pieces, others one by one: both against the plain form
    wide = logits(6, E + 8, dtype, seed=E)
    bias = 0.2 * logits(1, E + 4, seed=3)[0]
    avail = torch.rand(E, generator=torch.Generator().manual_seed(1)).cuda() < 0.8
    for off in (0, 1, 2, 8):
        z = wide[:, off:off + E]
        for rule in (RouteRule(6, "sigmoid", G, max(1, G // 2), scale=2.5), RouteRule(6, "softmax", G, max(1, G // 2), 1, False)):
            check(z, rule)
            check(z, rule, bias=bias[off // 2:off // 2 + E], available=avail)


def test_streams_and_graphs():
    z = logits(300, 256, seed=8)
    rule = RouteRule(8, "sigmoid", 8, 4, scale=2.5)
    bias = 0.1 * logits(1, 256, seed=9)[0]
    want = route_scored(z, rule, bias=bias)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = route_scored(z, rule, bias=bias, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    buf = z.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = route_scored(buf, rule, bias=bias)
    for seed in (20, 21):
        new = logits(300, 256, seed=seed)
        buf.copy_(new)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(route_scored(new, rule, bias=bias), out))


def test_refusals():
    z = logits(2, 64)
    with pytest.raises(_lib.YanahError):
        route_scored(z, RouteRule(65))
    with pytest.raises(_lib.YanahError):
        route_scored(z, RouteRule(4, n_groups=7, top_groups=2))
    with pytest.raises(_lib.YanahError):
        route_scored(z, RouteRule(17, n_groups=8, top_groups=2))
    with pytest.raises(ValueError):
        route_scored(z, RouteRule(4), bias=torch.zeros(63, device="cuda"))
    with pytest.raises(TypeError):
        route_scored(z, RouteRule(4), bias=torch.zeros(64, device="cuda", dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        route_scored(z, RouteRule(4), bias=torch.zeros(64))
    with pytest.raises(RuntimeError):
        route_scored(z.clone().requires_grad_(), RouteRule(4))
