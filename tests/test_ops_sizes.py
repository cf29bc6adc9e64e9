"""Sizes at the border of what the operators take, decided on the host (these run without a GPU)."""
from __future__ import annotations

import pytest

pytest.importorskip("torch")

from tests.test_ops_refusals import INV, experts
from yanah_b200 import _lib


@pytest.mark.parametrize("k", [1, 3, 32])
def test_pairs_of_rows_and_experts(k):
    # rows * top_k is not formed: it would pass 64 bits
    for rows in ((1 << 22) // k + 1, 1 << 40, (1 << 59) + 1, (1 << 62) + 2, (1 << 63) - 1):
        assert experts(rows=rows, k=k) == INV, rows


def test_rows_without_a_workspace():
    # those that go to the kernel which makes the codes itself, whatever the number of channels
    ws = _lib.lib().yn_i8_linear_ws_bytes
    for rows, k in ((1, 1), (1, 4096), (1, 98304), (2, 2560), (3, 2048), (3, 7)):
        assert ws(rows, k) == 0, (rows, k)
    for rows, k in ((1, 98305), (2, 4096), (3, 2049), (4, 1), (3, 4096)):
        assert ws(rows, k) >= rows * k, (rows, k)


def test_pointers_that_are_not_aligned_to_their_elements():
    # a kernel would fault on them
    import ctypes as C

    from tests.test_ops_refusals import P, mat, rule
    lib, odd, half = _lib.lib(), C.c_void_p(257), C.c_void_p(258)
    r = rule()

    def route(logits=P, dtype=0, bias=None, ids=P, w=P):
        return lib.yn_route_scored(C.byref(r), logits, dtype, 64, 2, bias, None, ids, w, None)

    for kw in (dict(logits=half), dict(logits=odd, dtype=1), dict(logits=odd, dtype=2), dict(bias=half), dict(ids=half), dict(w=odd)):
        assert route(**kw) == INV, kw

    def logprobs(at, p):
        a = [P] * 6
        a[at] = p
        return lib.yn_token_logprobs(P, 1, 100, 3, 100, a[0], 4, a[1], a[2], a[3], a[4], a[5], None)

    for at in range(6):
        assert logprobs(at, half) == INV, at
    assert lib.yn_i8_quant_rows(odd, 1, 64, 2, 64, P, 64, P, None) == INV
    assert lib.yn_i8_quant_rows(P, 1, 64, 2, 64, P, 64, half, None) == INV
    m = mat(scales=258)
    assert lib.yn_i8_linear(C.byref(m), P, 0, 64, 2, P, 0, 32, None, 0, None) == INV
    g, d = mat(4, 32, 64, 64, 2048, 32), mat(4, 64, 32, 32, 2048, 64)

    def experts_err(x=P, ids=P, w=P, res=None, out=P, err=None):
        return lib.yn_i8_experts_err(C.byref(g), C.byref(g), C.byref(d), x, 1, 64, 2, ids, w, 2, res, 64, out, 64, P, 1 << 30,
                                     err, None)

    for kw in (dict(x=odd), dict(ids=half), dict(w=half), dict(res=odd), dict(out=odd), dict(err=half)):
        assert experts_err(**kw) == INV, kw


def test_strides_of_matrices_that_are_not_in_order():
    # a tensor map whose strides are not multiples of one another reads past the matrices
    from tests.test_ops_refusals import mat
    UNS = _lib.YN_E_UNSUPPORTED
    ok = mat(4, 32, 64, 64, 2048, 32)
    d = mat(4, 64, 32, 32, 2048, 64)
    for ms, rs in ((2048 + 16, 64), (2048 - 64, 64), (2000, 80), (64, 64 * 3), (80, 320 + 80 + 16), (96, 64 * 4)):
        bad = mat(4, 32, 64, rs, ms, 32)
        assert experts(g=bad, u=ok, d=d) == UNS and experts(g=ok, u=bad, d=d) == UNS, (ms, rs)
        assert experts(g=ok, u=ok, d=mat(4, 64, 32, rs, ms, 64)) == (UNS if (ms, rs) != (2048 - 64, 64) else UNS)
    # matrices that overlap
    for m in (mat(4, 32, 64, 64, 48, 32), mat(4, 32, 64, 64, 2048, 31)):
        assert experts(g=m, u=ok, d=d) == INV
