"""GPU test of the operators' refusals on a stream that is given: the same as on the current one."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from yanah_b200.int8 import Int8Matrix, int8_experts, int8_linear
from yanah_b200.logprobs import token_logprobs
from yanah_b200.routing import RouteRule, route_scored

pytestmark = pytest.mark.gpu


def test_tensors_of_the_cpu_are_refused_alike():
    z, cpu = torch.randn(3, 64, device="cuda"), torch.zeros(64)
    rule = RouteRule(2)
    ids, w = route_scored(z, rule)
    m = Int8Matrix(torch.zeros(4, 64, 64, dtype=torch.int8, device="cuda"), torch.zeros(4, 64, device="cuda"))
    host = Int8Matrix(m.codes.cpu(), m.scales.cpu())
    calls = [lambda s: route_scored(z, rule, cpu, stream=s),
             lambda s: token_logprobs(z, torch.zeros(3, dtype=torch.int32), stream=s),
             lambda s: int8_linear(z, Int8Matrix(host.codes[0], host.scales[0]), stream=s),
             lambda s: int8_experts(z, ids, w, m, host, m, stream=s),
             lambda s: int8_experts(z, ids.cpu(), w, m, m, m, stream=s),
             lambda s: int8_experts(z, ids, w, m, m, m, residual=z.cpu(), stream=s)]
    for call in calls:
        for stream in (None, torch.cuda.Stream()):
            with pytest.raises(ValueError):
                call(stream)
