"""GPU tests of the device grouping's answer to ids that name no expert."""
from __future__ import annotations

import ctypes as C

import pytest

torch = pytest.importorskip("torch")

from tests.gpu_helpers import small_config
from yanah_b200 import _lib
from yanah_b200.device import dims_struct, stream_ptr

pytestmark = pytest.mark.gpu

BAD_EXPERT = 2


def plan(name, ids):
    cfg = small_config(bits=(4, 4), gs=64, hidden=512, n_experts=16, top_k=2, inter=512, shared=0, seed=7)
    d, T, lib = dims_struct(cfg), ids.shape[0], _lib.lib()
    up, dn = C.c_int32(0), C.c_int32(0)
    _lib.check(lib.yn_prefill_max_tiles(C.byref(d), T, C.byref(up), C.byref(dn)))
    new = lambda *s: torch.full(s, -5, dtype=torch.int32, device="cuda")
    row, of, tu, td, n, err = new(2 * T), new(T, 2), new(up.value, 4), new(dn.value, 4), new(2), torch.zeros(1, dtype=torch.int32, device="cuda")
    _lib.check(getattr(lib, name)(C.byref(d), ids.data_ptr(), T, row.data_ptr(), of.data_ptr(), tu.data_ptr(), up.value,
                                  td.data_ptr(), dn.value, n.data_ptr(), err.data_ptr(), stream_ptr()))
    torch.cuda.synchronize()
    return of.cpu(), n.cpu(), err.item()


@pytest.mark.parametrize("bad", [None, -1, -2, 16])
def test_an_id_without_an_expert(bad):
    ids = torch.arange(24, dtype=torch.int32).view(12, 2) % 16
    if bad is not None:
        ids[3, 1] = bad
    ids = ids.cuda()
    of, n, err = plan("yn_prefill_plan", ids)
    assert err == (BAD_EXPERT if bad is not None else 0)     # softmax top-k leaves no column empty: -1 is an error
    by_rule, rn, rerr = plan("yn_prefill_plan_by_rule", ids)
    assert rerr == (BAD_EXPERT if bad in (-2, 16) else 0)
    for p in (of, by_rule):
        assert sorted(p[p >= 0].tolist()) == list(range(24 if bad is None else 23))
        assert bad is None or p[3, 1] == -1
    assert torch.equal(n, rn)
