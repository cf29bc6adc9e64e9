"""Refusals of the scored router, the 8-bit products and the token log probabilities that
happen on the host, before any device work (these run without a GPU)."""
from __future__ import annotations

import ctypes as C

import pytest

torch = pytest.importorskip("torch")

from yanah_b200 import _lib
from yanah_b200.int8 import Int8Matrix, int8_experts, int8_linear, quantize_rows
from yanah_b200.logprobs import token_logprobs
from yanah_b200.routing import RouteRule, route_scored
from yanah_b200.speculation import verify_rows

INV, UNS = _lib.YN_E_INVALID, _lib.YN_E_UNSUPPORTED
P = C.c_void_p(256)   # never dereferenced: every call below is refused on the host


def route(rule, logits=P, dtype=0, stride=None, rows=2, ids=P, w=P):
    return _lib.lib().yn_route_scored(C.byref(rule), logits, dtype, rule.n_experts if stride is None else stride, rows, None,
                                      None, ids, w, None)


def rule(E=64, k=4, score=0, G=1, kept=1, gt=2, norm=1, scale=1.0):
    return _lib.RouteRuleStruct(E, k, score, G, kept, gt, norm, scale)


def test_route_scored():
    for bad, rc in ((rule(E=0), INV), (rule(k=0), INV), (rule(k=65), INV), (rule(E=1025), UNS), (rule(k=32), UNS),
                    (rule(score=2), INV), (rule(G=0), INV), (rule(G=7), INV), (rule(G=8, kept=9), INV),
                    (rule(G=8, kept=0), INV), (rule(G=64, kept=4), UNS), (rule(gt=3), INV), (rule(k=9, G=8, kept=1), INV)):
        assert route(bad) == rc
    assert route(rule(), dtype=3) == INV and route(rule(), stride=63) == INV and route(rule(), rows=-1) == INV
    assert route(rule(), logits=None) == INV and route(rule(), ids=None) == INV
    assert route(rule(), rows=0, logits=None) == _lib.YN_OK
    with pytest.raises(ValueError):
        RouteRule(4, "tanh")


def logprobs(dtype=0, stride=100, rows=3, vocab=100, tokens=P, n=0, top=P, logits=P, lp=P):
    return _lib.lib().yn_token_logprobs(logits, dtype, stride, rows, vocab, tokens, n, lp, P, P, top, top, None)


def test_token_logprobs():
    for kw in (dict(dtype=5), dict(stride=99), dict(vocab=0), dict(n=-1), dict(n=65), dict(vocab=3, n=4), dict(n=3, top=None),
               dict(logits=None), dict(lp=None), dict(rows=-1), dict(logits=C.c_void_p(258))):
        assert logprobs(**kw) == INV, kw
    assert logprobs(vocab=2 ** 31, stride=2 ** 31) == UNS
    assert logprobs(rows=0, logits=None) == _lib.YN_OK


def mat(mats=1, rows=32, cols=64, rs=64, ms=2048, ss=32, codes=256, scales=256):
    return _lib.I8Mat(codes, scales, rs, ms, ss, mats, rows, cols)


def linear(m, dtype=0, xs=64, rows=2, ys=32, x=P, y=P, ws=None, nb=0):
    return _lib.lib().yn_i8_linear(C.byref(m), x, dtype, xs, rows, y, 0, ys, ws, nb, None)


def test_int8_linear():
    for m, rc in ((mat(codes=None), INV), (mat(scales=None), INV), (mat(rows=0), INV), (mat(cols=0), INV), (mat(codes=264), INV),
                  (mat(rs=72), INV), (mat(rs=48), INV), (mat(mats=2), INV), (mat(mats=2, ms=2056), INV),
                  (mat(cols=131073, rs=131088), UNS), (mat(rs=1 << 40), UNS)):
        assert linear(m) == rc
    for kw in (dict(dtype=4), dict(xs=63), dict(ys=31), dict(rows=-1), dict(x=None), dict(y=None), dict(x=C.c_void_p(258)),
               dict(rows=20), dict(rows=20, ws=P, nb=64)):
        assert linear(mat(), **kw) == INV, kw
    assert linear(mat(), rows=0, x=None) == _lib.YN_OK
    assert _lib.lib().yn_i8_linear_ws_bytes(1, 2048) == 0 and _lib.lib().yn_i8_linear_ws_bytes(9, 2048) >= 9 * 2048
    q = _lib.lib().yn_i8_quant_rows
    assert q(P, 0, 63, 2, 64, P, 64, P, None) == INV and q(P, 0, 64, 2, 64, P, 63, P, None) == INV
    assert q(P, 9, 64, 2, 64, P, 64, P, None) == INV and q(None, 0, 64, 2, 64, P, 64, P, None) == INV
    assert q(None, 0, 64, 0, 64, None, 64, None, None) == _lib.YN_OK


def experts(g=None, u=None, d=None, rows=2, k=2, dtype=1, xs=64, ids=P, ws=P, nb=1 << 30, res=None, rs=0, x=P):
    g = g or mat(4, 32, 64, 64, 2048, 32)
    u = u or mat(4, 32, 64, 64, 2048, 32)
    d = d or mat(4, 64, 32, 32, 2048, 64)
    return _lib.lib().yn_i8_experts(C.byref(g), C.byref(u), C.byref(d), x, dtype, xs, rows, ids, P, k, res, rs, P, 64, ws, nb,
                                    None)


def test_int8_experts():
    for kw in (dict(u=mat(3, 32, 64, 64, 2048, 32)), dict(d=mat(4, 64, 64, 64, 4096, 64)), dict(dtype=7), dict(xs=63), dict(ids=None),
               dict(ws=None), dict(nb=16), dict(ws=C.c_void_p(128)), dict(res=P, rs=63), dict(rows=-1), dict(rows=1 << 22),
               dict(x=C.c_void_p(257))):
        assert experts(**kw) == INV, kw
    assert experts(k=33) == UNS and experts(k=0) == UNS
    assert experts(rows=0, x=None) == _lib.YN_OK
    assert _lib.lib().yn_i8_experts_ws_bytes(0, 4, 8, 64, 64, 1) == 0


def test_tensors_of_the_cpu_are_refused():
    z = torch.zeros(2, 64)
    w = Int8Matrix(torch.zeros(8, 64, dtype=torch.int8), torch.zeros(8))
    for call in (lambda: route_scored(z, RouteRule(4)), lambda: token_logprobs(z), lambda: quantize_rows(z),
                 lambda: int8_linear(z, w), lambda: int8_experts(z, z.int(), z, w, w, w)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: route_scored(z.double(), RouteRule(4)), lambda: token_logprobs(z.int()), lambda: quantize_rows(z.long())):
        with pytest.raises(TypeError):
            call()
    with pytest.raises(ValueError):
        verify_rows(z, w, torch.zeros(4, dtype=torch.int32))
    with pytest.raises(ValueError):
        verify_rows(z, w, torch.zeros(1, dtype=torch.int32), n_top=0)


def test_arguments_that_require_a_gradient_are_refused():
    # no operator has a backward pass: a gradient is refused, not dropped (-1: the index of the CPU)
    from yanah_b200.int8 import _mat
    from yanah_b200.launch import check_like
    w = torch.zeros(3, 2, requires_grad=True)
    with pytest.raises(RuntimeError, match="weights requires a gradient"):
        check_like(w, -1, (3, 2), (torch.float32,), "weights")
    m = Int8Matrix(torch.zeros(8, 64, dtype=torch.int8), torch.zeros(8, requires_grad=True))
    with pytest.raises(RuntimeError, match="w's scales requires a gradient"):
        _mat(m, -1, "w")
    with torch.no_grad():
        check_like(w, -1, (3, 2), (torch.float32,), "weights")
        assert _mat(m, -1, "w").rows == 8
