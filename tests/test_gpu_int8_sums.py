"""GPU tests of the sum over a row's 8-bit experts: it is made of fp32 products and rounded
once, for few pairs and for grouped ones, so that a row's answer is the same, bit for bit, in a
batch of any size.

Tolerance against 64 bits, for two experts that differ in their down scales alone: both have the
same activations, so that a moved code of one moves in the other too and leaves the share
|w0 s0 + w1 s1| of it, inside 4e-3 of the sum. A product is a conversion, two factors, a row scale of
two roundings and one fused step, each 2^-24: below 2^-21 of the product, 2^-20 asked. The output's
rounding is eps / 2.
"""
from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from tests import ref64
from tests.test_gpu_int8 import DTS, np64, setup
from yanah_b200.int8 import Int8Matrix, int8_experts

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTS)
def test_a_row_is_the_same_in_a_batch_of_any_size(dtype):
    # 1, 2 and 16 rows of 4 pairs go to the kernels of few pairs, 17 and more are grouped
    x, ids, w, mats, res = setup(24, 333, 712, 200, 4, dtype, seed=31, absent=0.1)
    for residual in (res, None):
        def run(lo, hi):
            return int8_experts(x[lo:hi], ids[lo:hi], w[lo:hi], *mats,
                                residual=None if residual is None else residual[lo:hi])
        whole = run(0, 200)
        for lo, n in ((0, 1), (57, 1), (199, 1), (11, 2), (64, 16), (100, 17), (30, 100)):
            assert torch.equal(run(lo, lo + n), whole[lo:lo + n]), (lo, n)


@pytest.mark.parametrize("dtype", DTS[:2])
@pytest.mark.parametrize("T", [2, 60])
def test_the_sum_is_rounded_once(T, dtype):
    # the same values in fp32 have the same codes: their sum, rounded, is the answer
    x, ids, w, mats, res = setup(16, 160, 256, T, 4, dtype, seed=32)
    for r in (None, res):
        got = int8_experts(x, ids, w, *mats, residual=r)
        want = int8_experts(x.float(), ids, w, *mats, residual=None if r is None else r.float())
        assert torch.equal(got, want.to(dtype))


@pytest.mark.parametrize("dtype", DTS)
@pytest.mark.parametrize("T", [3, 40, 300])
def test_products_that_cancel(T, dtype):
    x, ids, w, mats, _ = setup(2, 128, 256, T, 2, dtype, seed=33)
    for m in mats:
        m.codes[1] = m.codes[0]
        m.scales[1] = m.scales[0]
    mats[2].scales[1] = 1.01 * mats[2].scales[0]
    ids[:, 0], ids[:, 1] = 0, 1
    w[:, 0], w[:, 1] = 64.0, -63.36               # 64 - 63.36 * 1.01 = 0.0064: 1e-4 of a product is left
    got = np64(int8_experts(x, ids, w, *mats))
    m = [(np64(a.codes), np64(a.scales)) for a in mats]
    one = [ref64.experts(np64(x), ids[:, j:j + 1].cpu().numpy(), np64(w[:, j:j + 1]), *m) for j in range(2)]
    want, size = one[0] + one[1], np.abs(one[0]) + np.abs(one[1])
    assert np.linalg.norm(want) <= 2e-4 * np.linalg.norm(one[0])
    norm = np.linalg.norm
    assert norm(got - want) <= (4e-3 + torch.finfo(dtype).eps / 2) * norm(want) + 2.0 ** -20 * norm(size)


@pytest.mark.parametrize("dtype", DTS)
@pytest.mark.parametrize("T", [3, 60])
def test_the_output_may_be_the_residual(T, dtype):
    x, ids, w, mats, res = setup(16, 96, 257, T, 4, dtype, seed=34)
    want = int8_experts(x, ids, w, *mats, residual=res)
    wide = torch.full((T, 300), 7.0, dtype=dtype, device="cuda")
    for place in (wide[:, 8:265], wide[:, 5:262], res):
        place.copy_(res)
        assert int8_experts(x, ids, w, *mats, residual=place, out=place) is place
        assert torch.equal(place, want)
        if place is not res:
            place.fill_(7.0)
            assert (wide == 7.0).all()
