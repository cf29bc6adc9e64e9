"""GPU tests of the scored router's order where every score of a row is far below 1.

The kernel takes 2^(z log2 e) in fp32, so that a score of e^z is off by up to 2^-24 |z|, from the
rounding of the exponent, beside a few ulp. Rows are built whose fp32 order is wrong by that: near
z = -50 the scores that a rounded exponent makes larger stand against ones that it makes smaller, and
a bias gives the second a lead of 2e-7 of a score in 64-bit arithmetic. The ids are those of the 64-bit
form, without a tolerance.
"""
from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from tests import ref64
from yanah_b200.routing import RouteRule, route_scored

pytestmark = pytest.mark.gpu

LEAD = 2e-7


def off(z):
    """Relative error of 2^fl(z log2 e) against e^z."""
    y = (z * np.float32(1.4426950408889634)).astype(np.float64)
    return np.expm1(y * np.log(2.0) - z.astype(np.float64))


def low_logits(rng, low, high, n):
    """Logits whose fp32 scores come out too large and too small, n of each."""
    z = rng.uniform(low, high, 400 * n).astype(np.float32)
    order = np.argsort(off(z))
    return z[order[-n:]], z[order[:n]]


def lift(small, large):
    """Biases (fp32) that bring the sums of scores of `small` a little above those of `large`."""
    a, b = (np.exp(v.astype(np.float64)).sum(-1) for v in (large, small))
    return (a * (1 + LEAD) - b).astype(np.float32)


def route(z, rule, bias):
    """Every row with a bias of its own: a call for each."""
    ids = [route_scored(z[i:i + 1], rule, bias[i])[0] for i in range(len(z))]
    return torch.cat(ids).cpu().numpy()


@pytest.mark.parametrize("low,high", [(-62.0, -61.9), (-50.0, -49.9), (-31.1, -31.0)])
def test_neighbours(low, high):
    rng, n, E = np.random.default_rng(5), 60, 64
    large, small = low_logits(rng, low, high, n)
    z = np.full((n, E), -np.inf, np.float32)
    bias = np.zeros((n, E), np.float32)
    z[:, 7], z[:, 40] = large, small
    bias[:, 40] = lift(small[:, None], large[:, None])
    got = route(torch.from_numpy(z).cuda(), RouteRule(2, "sigmoid"), torch.from_numpy(bias).cuda())
    for i in range(n):
        want, _ = ref64.route(z[i:i + 1], 2, "sigmoid", bias[i])
        assert want[0].tolist() == [40, 7]
        assert got[i].tolist() == want[0].tolist(), (i, z[i, [7, 40]], bias[i, 40])


@pytest.mark.parametrize("low,high", [(-62.0, -61.9), (-50.0, -49.9), (-31.1, -31.0)])
@pytest.mark.parametrize("E", [64, 72])
def test_groups(E, low, high):
    # the best group by the sum of its two best: four errors of the same direction
    rng, n = np.random.default_rng(6), 60
    large, small = low_logits(rng, low, high, 2 * n)
    large, small = large.reshape(n, 2), small.reshape(n, 2)
    z = np.full((n, E), -np.inf, np.float32)
    bias = np.zeros((n, E), np.float32)
    per = E // 8
    z[:, [per, per + 3]], z[:, [5 * per + 1, 5 * per + 2]] = large, small
    bias[:, 5 * per + 1] = lift(small, large)
    got = route(torch.from_numpy(z).cuda(), RouteRule(2, "sigmoid", n_groups=8, top_groups=1), torch.from_numpy(bias).cuda())
    for i in range(n):
        want, _ = ref64.route(z[i:i + 1], 2, "sigmoid", bias[i], groups=8, kept=1)
        assert set(want[0].tolist()) == {5 * per + 1, 5 * per + 2}
        assert got[i].tolist() == want[0].tolist(), (i, z[i][z[i] > -np.inf], bias[i].max())
