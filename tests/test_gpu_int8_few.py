"""GPU tests of the 8-bit products at the borders between the kernel of few rows and the tensor
cores: a row's answer does not depend on which of them made it."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from tests.test_gpu_int8 import DTS, check_linear, matrix, normal
from yanah_b200.int8 import int8_linear

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTS)
@pytest.mark.parametrize("K,N", [(2048, 4096), (2048, 4100), (2048, 8192), (2048, 8196), (2049, 8300), (4096, 4099),
                                 (8192, 1025), (12288, 700), (8200, 130), (98304, 5), (98305, 5), (1000, 20001)])
def test_borders_of_the_few_rows(K, N, dtype):
    x, w = normal(7, K, seed=K, dtype=dtype), matrix(N, cols=K, seed=N)
    whole = check_linear(x, w, torch.float32)
    for T in (1, 2, 3, 4, 5, 6):
        assert torch.equal(int8_linear(x[:T], w, torch.float32), whole[:T])
        assert torch.equal(int8_linear(x[7 - T:], w, torch.float32), whole[7 - T:])
