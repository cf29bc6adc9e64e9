"""GPU tests of who learns of an error of the 8-bit products: a stack, or a call with an error word
of its own, has it there; all other calls on a device share one word."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from tests.gpu_helpers import bf16_dev, hidden_rows, small_config
from tests.test_gpu_int8 import setup
from yanah_b200.int8 import check_error, int8_experts
from yanah_b200.prefill import PrefillStack

pytestmark = pytest.mark.gpu

BAD_EXPERT = 2


def bad_call(T, **kw):
    x, ids, w, mats, res = setup(16, 96, 256, T, 4, seed=3)
    ids[1, 2] = 16
    return int8_experts(x, ids, w, *mats, residual=res, **kw)


@pytest.mark.parametrize("T", [2, 90])
def test_a_stack_does_not_report_the_errors_of_others(T):
    cfg = small_config(bits=(4, 4), gs=64, hidden=512, n_experts=16, top_k=2, inter=512, shared=0, seed=7)
    stacks = [PrefillStack(cfg, max_rows=8, experts="int8", layers=[0]) for _ in range(2)]
    h = bf16_dev(hidden_rows(cfg, 8, stream=3))
    bad_call(T)
    out = [st.prefill(h).clone() for st in stacks]
    assert [st.check_error() for st in stacks] == [0, 0]
    assert check_error() == BAD_EXPERT and check_error() == 0
    # a stack's own errors are its own, and one check clears all of its words
    stacks[0].err.fill_(BAD_EXPERT)
    stacks[0].route_ws[:4].view(torch.int32).fill_(1)
    assert stacks[1].check_error() == 0 and check_error() == 0
    assert stacks[0].check_error() == BAD_EXPERT and stacks[0].check_error() == 0
    assert torch.equal(out[0], out[1])


@pytest.mark.parametrize("T", [2, 90])
def test_an_error_word_of_the_callers_own(T):
    mine, other = (torch.zeros(1, dtype=torch.int32, device="cuda") for _ in range(2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    want = bad_call(T)
    assert check_error() == BAD_EXPERT
    for stream in (None, side):
        mine.zero_()
        side.wait_stream(torch.cuda.current_stream())
        got = bad_call(T, err=mine, stream=stream)
        torch.cuda.synchronize()
        assert mine.item() == BAD_EXPERT and other.item() == 0 and check_error() == 0
        assert torch.equal(got, want)
    for bad in (mine.long(), torch.zeros(2, dtype=torch.int32, device="cuda"), mine.cpu()):
        with pytest.raises((TypeError, ValueError)):
            bad_call(T, err=bad)


def test_no_error_is_lost_between_reading_and_clearing():
    # a check on one stream while a call on another sets the word: the check, or the one after it, has it
    x, ids, w, mats, res = setup(16, 96, 256, 2, 4, seed=3)
    ids[1, 2] = 16
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    assert check_error() == 0
    for n in range(1500):
        with torch.cuda.stream(side):
            torch.cuda._sleep(20000 + 1000 * (n % 100))   # 10 to 60 us, so that the call meets every part of the check
            int8_experts(x, ids, w, *mats, residual=res)
        seen = check_error()
        side.synchronize()
        assert seen == BAD_EXPERT or check_error() == BAD_EXPERT, n
