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
