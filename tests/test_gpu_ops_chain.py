"""The scored router, the 8-bit experts and the token log probabilities as the framework
uses them together: a prompt pass and a verify pass, and the backend's routing by a rule.

Bounds: the 8-bit matrices lie within half a step of the dequantised records, value by
value; a layer on them is compared with the 64-bit form on the same matrices, within the
bound of the experts' own tests (4e-3 of the experts' part plus half a bf16 step).
"""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import cpu
from tests import ref64
from tests.gpu_helpers import bf16_dev, bf16_np, hidden_rows, rel_l2, small_config
from yanah_b200 import _lib
from yanah_b200.device import stream_ptr
from yanah_b200.int8 import int8_experts, int8_linear, quantize_rows
from yanah_b200.logprobs import token_logprobs
from yanah_b200.prefill import PrefillStack
from yanah_b200.routing import RouteRule
from yanah_b200.speculation import verify_rows

pytestmark = pytest.mark.gpu


def config():
    return small_config(bits=(4, 4), gs=64, hidden=512, n_experts=16, top_k=2, inter=512, shared=0, seed=7)


def test_int8_prompt_pass():
    cfg, T = config(), 60
    h = bf16_dev(hidden_rows(cfg, T, stream=3))
    rec = PrefillStack(cfg, max_rows=T)
    i8 = PrefillStack(cfg, max_rows=T, experts="int8")
    # the matrices: each value within half a step of the record's
    spec = cfg.record_spec(1)
    for part, m in enumerate(i8.int8[1]):
        e, rows, cols = m.codes.shape
        for i in (0, e - 1):
            full = torch.empty(rows, cols, device="cuda")
            base = rec.arenas[1].base + i * rec.arenas[1].slot_bytes
            q = _lib.QMat(*(base + spec.offsets[3 * part + j] for j in range(3)), rows, cols, spec.bits, spec.group_size)
            _lib.check(_lib.lib().yn_dequantize(C.byref(q), full.data_ptr(), stream_ptr()))
            torch.cuda.synchronize()
            step = m.scales[i].double().unsqueeze(1)
            # half a step, and the rounding of the scale (2^-24) times a code of at most 127
            assert ((m.codes[i].double() * step - full.double()).abs() <= step * (0.5 + 127 * 2 ** -24)).all()
            assert (m.codes[i].abs().amax(1) == 127).all()
    for layer in (0, 1):
        m = [(x.codes.cpu().numpy(), x.scales.cpu().numpy()) for x in i8.int8[layer]]
        for n in (1, 7, T):
            a, b = torch.empty_like(h[:n]), torch.empty_like(h[:n])
            rec.layer(layer, h[:n], a)
            i8.layer(layer, h[:n], b)
            torch.cuda.synchronize()
            assert torch.equal(rec.ids[:n], i8.ids[:n]) and torch.equal(rec.w[:n], i8.w[:n])
            res = h[:n].double().cpu().numpy()
            want = ref64.experts(i8.x[:n].double().cpu().numpy(), i8.ids[:n].cpu().numpy(), i8.w[:n].cpu().numpy(), *m,
                                 residual=res)
            err = np.linalg.norm(b.double().cpu().numpy() - want)
            assert err <= 4e-3 * np.linalg.norm(want - res) + 2 ** -8 * np.linalg.norm(want)
    assert rec.check_error() == 0 and i8.check_error() == 0
    assert i8.prefill(h).shape == (T, cfg.hidden)
    with pytest.raises(ValueError):
        i8.plan(T)


@pytest.mark.parametrize("experts", ["records", "int8"])
def test_prompt_pass_by_a_rule(experts):
    cfg, T = config(), 45
    rule = RouteRule(2, "sigmoid", n_groups=4, top_groups=2, scale=1.5)
    bias = 0.3 * torch.randn(cfg.n_layers, cfg.n_experts, generator=torch.Generator().manual_seed(2)).cuda()
    st = PrefillStack(cfg, max_rows=T, rule=rule, choice_bias=bias, experts=experts)
    h = bf16_dev(hidden_rows(cfg, T, stream=4))
    out = torch.empty_like(h)
    st.layer(1, h, out)
    torch.cuda.synchronize()
    assert st.check_error() == 0
    logits = cpu.OracleStack(cfg, threads=8).post_attention(1, bf16_np(h))["logits"]
    ids, w = ref64.route(logits, 2, "sigmoid", bias[1].cpu().numpy(), groups=4, kept=2, scale=1.5)
    assert np.array_equal(st.ids[:T].cpu().numpy(), ids)
    assert np.allclose(st.w[:T].cpu().numpy(), w, rtol=4e-6)
    with pytest.raises(ValueError):
        PrefillStack(cfg, max_rows=4, rule=RouteRule(3))
    with pytest.raises(ValueError):
        PrefillStack(cfg, max_rows=4, experts="int4")


@pytest.mark.parametrize("T", [1, 5, 40])
def test_backend_routes_by_a_rule(T):
    from yanah_b200.backend import CudaMoEBackend
    from yanah_b200.device import fill_synthetic_experts
    cfg = config()
    rule = RouteRule(2, "sigmoid", scale=2.0)
    bias = 0.3 * torch.randn(cfg.n_layers, cfg.n_experts, generator=torch.Generator().manual_seed(2)).cuda()
    be = CudaMoEBackend(cfg, "cuda", rule=rule, choice_bias=bias)
    plain = CudaMoEBackend(cfg, "cuda")
    mem = be.make_expert_memory(cfg.n_experts)
    fill_synthetic_experts(mem.arena, cfg, 0)
    h = bf16_dev(hidden_rows(cfg, T, stream=5))
    h_res, x, logits = be.pre_moe(0, h)
    ids, w = be.route(logits)
    oracle = cpu.OracleStack(cfg, threads=8)
    pa = oracle.post_attention(0, bf16_np(h))
    ri, rw = ref64.route(pa["logits"], 2, "sigmoid", bias[0].cpu().numpy(), scale=2.0)
    assert np.array_equal(ids, ri)
    assert np.allclose(w.cpu().numpy(), rw, rtol=4e-6)
    out = be.moe(0, x, ids, w, mem, {e: e for e in range(cfg.n_experts)})
    # the routed experts of row 0 with these weights
    ref = sum(float(rw[0, j]) * cpu.bf16_to_f32(oracle.expert(0, int(ri[0, j]), pa["x"][0])[1]) for j in range(2))
    got = out[0].double().cpu().numpy()
    assert np.linalg.norm(got - ref) <= 1e-2 * np.linalg.norm(ref)
    assert be.check_error() == 0
    # a backend without a rule is as it was
    plain.pre_moe(0, h)
    pi, pw = plain.route(None)
    assert np.array_equal(pi, pa["ids"]) and np.array_equal(pw.cpu().numpy(), pa["w"])


def test_verify_rows():
    V, H, d = 5003, 512, 4
    g = torch.Generator().manual_seed(9)
    head = quantize_rows((torch.randn(V, H, generator=g) / H ** 0.5).bfloat16().cuda())
    rows = (4 * torch.randn(1 + d, H, generator=g)).bfloat16().cuda()
    logits = int8_linear(rows, head, out_dtype=torch.float32)
    z = logits.double().cpu().numpy()
    want = ref64.linear(rows.double().cpu().numpy(), head.codes.cpu().numpy(), head.scales.cpu().numpy())
    assert np.abs(z - want).max() <= 2 ** -21 * np.abs(want).max()
    greedy = z.argmax(1)
    for n_ok in range(d + 1):
        draft = torch.tensor(greedy[:d], dtype=torch.int32)
        if n_ok < d:
            draft[n_ok] = (draft[n_ok] + 1) % V
        a = verify_rows(rows, head, draft.cuda(), n_top=5)
        assert a.accepted.item() == n_ok and a.next_token.item() == greedy[n_ok]
        ref = ref64.logprobs(z, draft.tolist() + [-1], 5)
        assert np.array_equal(a.answers.rank.cpu().numpy(), ref["rank"])
        assert np.array_equal(a.answers.top_ids.cpu().numpy(), ref["top_ids"])
        assert np.allclose(a.answers.logprob[:d].cpu().numpy(), ref["logprob"][:d], rtol=1e-5)
        assert torch.isnan(a.answers.logprob[d])
    none = verify_rows(rows[:1], head, torch.empty(0, dtype=torch.int32, device="cuda"))
    assert none.accepted.item() == 0 and none.next_token.item() == greedy[0]
    with pytest.raises(ValueError):
        verify_rows(rows, head, draft[:2].cuda())


def test_a_prompt_pass_answers_in_one_graph():
    # rows -> router by a rule -> 8-bit experts, two layers -> LM head -> log probabilities, captured and replayed
    cfg, T, V = config(), 33, 3001
    st = PrefillStack(cfg, max_rows=T, rule=RouteRule(2, "sigmoid"), experts="int8")
    head = quantize_rows((torch.randn(V, cfg.hidden, generator=torch.Generator().manual_seed(1)) * 1e-3).cuda())
    h = bf16_dev(hidden_rows(cfg, T, stream=6))
    tokens = torch.arange(T, dtype=torch.int32, device="cuda") * 7

    def run(rows):
        return token_logprobs(int8_linear(st.prefill(rows), head, out_dtype=torch.float32), tokens, n_top=4)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(h)
    torch.cuda.current_stream().wait_stream(side)
    buf = h.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(buf)
    for stream in (7, 8):
        new = bf16_dev(hidden_rows(cfg, T, stream=stream))
        want = [t.clone() for t in run(new)]
        buf.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, out))
    assert st.check_error() == 0


@pytest.mark.parametrize("experts", ["records", "int8"])
def test_rule_that_leaves_rows_short(experts):
    # a bias of -inf takes all experts but one, or all, out: the columns without an expert add nothing
    cfg, T = config(), 37
    bias = torch.full((cfg.n_layers, cfg.n_experts), -float("inf"), device="cuda")
    bias[0, 5] = 0.25
    st = PrefillStack(cfg, max_rows=T, rule=RouteRule(2, "sigmoid", scale=2.0), choice_bias=bias, experts=experts)
    h = bf16_dev(hidden_rows(cfg, T, stream=6))
    out = torch.full_like(h, float("nan"))
    for buf in (st.pair_of, st.pair_row):
        buf.fill_(0x7fffffff)       # what an allocation may hold
    st.layer(1, h, out)
    torch.cuda.synchronize()
    assert (st.ids[:T] == -1).all() and (st.w[:T] == 0).all() and torch.equal(out, h)
    st.layer(0, h, out)
    torch.cuda.synchronize()
    assert (st.ids[:T, 0] == 5).all() and (st.ids[:T, 1] == -1).all()
    # the weight: a quotient by a hardware reciprocal, 2 ulp, and its product with the scale
    assert ((st.w[:T, 0] - 2).abs() <= 4e-6).all() and (st.w[:T, 1] == 0).all() and st.check_error() == 0
    # expert 5 twice with weight 1 is the same sum (a + a = 2 a exactly)
    want = torch.empty_like(h)
    five, ones = torch.full((T, 2), 5, dtype=torch.int32, device="cuda"), torch.ones(T, 2, device="cuda")
    if experts == "int8":
        int8_experts(st.x[:T], five, ones, *st.int8[0], residual=h, out=want)
        torch.cuda.synchronize()
        # the same bf16 products, fp32 sums off by the weight's 2e-6, and the two roundings of half a step each
        a, b = out.double(), want.double()
        assert ((a - b).abs() <= 2 ** -7 * b.abs() + 4e-6 * (b - h.double()).abs()).all()
    else:
        y = cpu.OracleStack(cfg, threads=8)
        x = y.post_attention(0, bf16_np(h))["x"]
        for t in (0, T - 1):
            ref = cpu.bf16_to_f32(bf16_np(h)[t]) + 2.0 * cpu.bf16_to_f32(y.expert(0, 5, x[t])[1])
            got = out[t].double().cpu().numpy()
            assert np.linalg.norm(got - ref) <= 1e-2 * np.linalg.norm(ref)


def test_backend_refuses_rows_left_short():
    from yanah_b200.backend import CudaMoEBackend
    cfg = config()
    bias = torch.full((cfg.n_layers, cfg.n_experts), -float("inf"), device="cuda")
    be = CudaMoEBackend(cfg, "cuda", rule=RouteRule(2, "sigmoid"), choice_bias=bias)
    for T in (1, 40):
        be.pre_moe(0, bf16_dev(hidden_rows(cfg, T, stream=5)))
        with pytest.raises(RuntimeError, match="fewer than top_k"):
            be.route(None)
