"""Sizes at the border of what the operators take, decided on the host (these run without a GPU)."""
from __future__ import annotations

import pytest

pytest.importorskip("torch")

from tests.test_ops_refusals import INV, experts


@pytest.mark.parametrize("k", [1, 3, 32])
def test_pairs_of_rows_and_experts(k):
    # rows * top_k is not formed: it would pass 64 bits
    for rows in ((1 << 22) // k + 1, 1 << 40, (1 << 59) + 1, (1 << 62) + 2, (1 << 63) - 1):
        assert experts(rows=rows, k=k) == INV, rows
