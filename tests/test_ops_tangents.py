"""The operators have no forward-mode derivative: an argument with a tangent is refused, not
answered without one (the host's checks run without a GPU; -1 is the index of the CPU)."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")
from torch.autograd import forward_ad

from yanah_b200.int8 import Int8Matrix, _mat, int8_experts, int8_linear, quantize_rows
from yanah_b200.launch import check_like
from yanah_b200.logprobs import token_logprobs
from yanah_b200.routing import RouteRule, route_scored


def dual(t):
    return forward_ad.make_dual(t, torch.ones_like(t))


def test_checks():
    f32 = (torch.float32,)
    with forward_ad.dual_level():
        check_like(torch.zeros(3), -1, (3,), f32, "bias")
        with pytest.raises(RuntimeError, match="bias has a tangent"):
            check_like(dual(torch.zeros(3)), -1, (3,), f32, "bias")
        with torch.no_grad(), pytest.raises(RuntimeError, match="bias has a tangent"):
            check_like(dual(torch.zeros(3)), -1, (3,), f32, "bias")
        codes = torch.zeros(8, 64, dtype=torch.int8)
        assert _mat(Int8Matrix(codes, torch.zeros(8)), -1, "w").rows == 8
        with pytest.raises(RuntimeError, match="w's scales has a tangent"):
            _mat(Int8Matrix(codes, dual(torch.zeros(8))), -1, "w")


@pytest.mark.gpu
def test_operators():
    z, bias = torch.randn(3, 64, device="cuda"), torch.zeros(64, device="cuda")
    rule = RouteRule(2)
    ids, w = route_scored(z, rule)
    m = Int8Matrix(torch.zeros(4, 64, 64, dtype=torch.int8, device="cuda"), torch.zeros(4, 64, device="cuda"))
    one = Int8Matrix(m.codes[0], m.scales[0])
    with forward_ad.dual_level():
        calls = [lambda t, b: route_scored(t, rule, b), lambda t, b: token_logprobs(t), lambda t, b: quantize_rows(t),
                 lambda t, b: int8_linear(t, one), lambda t, b: int8_experts(t, ids % 4, w, m, m, m)]
        for call in calls:
            call(z, bias)
            with pytest.raises(RuntimeError, match="tangent"):
                call(dual(z), bias)
        with pytest.raises(RuntimeError, match="bias has a tangent"):
            calls[0](z, dual(bias))
        for kw in (dict(residual=dual(z)), dict(out=dual(z.clone()))):
            with pytest.raises(RuntimeError, match="tangent"):
                int8_experts(z, ids % 4, w, m, m, m, **kw)
        with pytest.raises(RuntimeError, match="weights has a tangent"):
            int8_experts(z, ids % 4, dual(w), m, m, m)
    route_scored(z, rule)
