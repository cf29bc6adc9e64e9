"""Options of the stacks that are refused where they are given, before any device work (these run
without a GPU), and the ones that a stack of some layers takes."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from tests.gpu_helpers import bf16_dev, hidden_rows, small_config
from yanah_b200.prefill import PrefillStack
from yanah_b200.routing import RouteRule

RULE = RouteRule(2, "sigmoid")


def config(shared=0):
    return small_config(bits=(4, 4, 4, 4), gs=64, hidden=512, n_experts=16, top_k=2, inter=512, shared=shared, seed=7)


def test_a_bias_has_a_row_for_each_layer():
    from yanah_b200.backend import CudaMoEBackend
    cfg = config()
    E = cfg.n_experts
    for make in (lambda bias, rule=RULE: PrefillStack(cfg, max_rows=4, layers=[1, 3], rule=rule, choice_bias=bias),
                 lambda bias, rule=RULE: CudaMoEBackend(cfg, rule=rule, choice_bias=bias)):
        for shape in ((3, E), (E,), (2, E + 1), (1, 2, E)):
            with pytest.raises(ValueError, match="choice_bias"):
                make(torch.zeros(shape))
        with pytest.raises(ValueError, match="needs a rule"):
            make(torch.zeros(2, E), None)
    # the model's biases are not those of a stack of two of its layers
    with pytest.raises(ValueError, match="row for each layer"):
        PrefillStack(cfg, max_rows=4, layers=[1, 3], rule=RULE, choice_bias=torch.zeros(cfg.n_layers, E))
    with pytest.raises(TypeError, match="choice_bias"):
        PrefillStack(cfg, max_rows=4, layers=[1, 3], rule=RULE, choice_bias=torch.zeros(2, E, dtype=torch.float64))


def test_8_bit_experts_refuse_a_configuration_with_a_shared_one():
    with pytest.raises(NotImplementedError, match="shared"):
        PrefillStack(config(shared=512), max_rows=4, experts="int8")


@pytest.mark.gpu
def test_the_biases_of_some_layers():
    cfg, T = config(), 9
    bias = 0.3 * torch.randn(cfg.n_layers, cfg.n_experts, generator=torch.Generator().manual_seed(2)).cuda()
    every = PrefillStack(cfg, max_rows=T, rule=RULE, choice_bias=bias)
    some = PrefillStack(cfg, max_rows=T, layers=[3, 1], rule=RULE, choice_bias=bias[[3, 1]])
    h = bf16_dev(hidden_rows(cfg, T, stream=4))
    a, b = torch.empty_like(h), torch.empty_like(h)
    for i, layer in enumerate((3, 1)):
        every.layer(layer, h, a)
        some.layer(i, h, b)
        torch.cuda.synchronize()
        assert torch.equal(every.ids[:T], some.ids[:T]) and torch.equal(every.w[:T], some.w[:T]) and torch.equal(a, b)


@pytest.mark.gpu
def test_8_bit_experts_refuse_events():
    # the list would stay empty
    cfg = config()
    st = PrefillStack(cfg, max_rows=4, layers=[0], experts="int8")
    h = bf16_dev(hidden_rows(cfg, 4, stream=4))
    for call in (lambda e: st.prefill(h, gemm_events=e), lambda e: st.layer(0, h, torch.empty_like(h), gemm_events=e)):
        with pytest.raises(ValueError, match="gemm_events"):
            call([])
    st.prefill(h)
    events = []
    PrefillStack(cfg, max_rows=4, layers=[0]).prefill(h, gemm_events=events)
    torch.cuda.synchronize()
    assert len(events) == 1 and events[0][0].elapsed_time(events[0][1]) > 0


@pytest.mark.gpu
def test_8_bit_experts_hold_no_buffers_of_the_records():
    cfg, T = config(), 2048
    K, H, I = cfg.top_k, cfg.hidden, cfg.moe_inter

    def asked():
        # what was asked of the allocator; memory_allocated counts its blocks, of which a large one may have up to 1 MiB more
        return torch.cuda.memory_stats()["requested_bytes.all.current"]

    def held(experts):
        before = asked()
        st = PrefillStack(cfg, max_rows=T, layers=[0], experts=experts)
        weights = sum(m.codes.untyped_storage().nbytes() + 4 * m.scales.numel() for m in st.int8[0]) if experts == "int8" \
            else st.arenas[0].buf.numel()
        return asked() - before - weights

    # x16 and y (pairs, H) and act (pairs, I), 16 bits each
    assert held("records") - held("int8") >= 2 * T * K * (2 * H + I)
