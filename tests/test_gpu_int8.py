"""GPU tests of the 8-bit integer products against a plain 64-bit implementation.

Codes are compared for equality, scales to one rounding (2^-24). A linear product: the
sum is exact, its conversion and two factors (one of them a rounded quotient) are four
roundings of 2^-24, and the output's rounding eps / 2: eps / 2 + 2^-21 of the value is
asked. Experts: the activations a are fp32 values of a hardware exponential and
reciprocal (a few ulp); where that moves one over the border between two codes the code is
off by one, so a product's error is at most sum_u |sd qd| sa over the moved ones. Expected
share of moved codes: the error in steps, below 127 * 8 * 2^-23 = 1.3e-4. The products'
rounding to bf16 before they are summed is half a step, 2^-8 = 3.9e-3, of each. Asked of
the whole output: relative 2-norm 4e-3 * (share of the experts' part in it <= 1) + eps / 2.
"""
from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from tests import ref64
from yanah_b200 import _lib
from yanah_b200.int8 import Int8Matrix, check_error, int8_experts, int8_linear, quantize_rows

pytestmark = pytest.mark.gpu
DTS = [torch.bfloat16, torch.float16, torch.float32]


def normal(*shape, seed=0, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(*shape, generator=g)).to(dtype).cuda()


def matrix(*lead, cols, seed=0, pad=0):
    g = torch.Generator().manual_seed(seed)
    st = (cols + 15) // 16 * 16 + pad
    codes = torch.zeros(*lead, st, dtype=torch.int8)[..., :cols]
    codes.copy_(torch.randn(*lead, cols, generator=g).mul(32).round().clamp(-127, 127))
    scales = (1 + torch.rand(*lead, generator=g)) / (32 * cols ** 0.5)
    st_codes = torch.zeros(*lead, st, dtype=torch.int8).cuda()
    st_codes[..., :cols] = codes.cuda()
    return Int8Matrix(st_codes[..., :cols], scales.cuda())


def np64(t):
    return t.double().cpu().numpy()


def check_linear(x, w, out_dtype=None):
    y = int8_linear(x, w, out_dtype)
    torch.cuda.synchronize()
    want = ref64.linear(np64(x), np64(w.codes), np64(w.scales))
    got = np64(y)
    tol = torch.finfo(y.dtype).eps / 2 + 2.0 ** -21
    tiny = torch.finfo(y.dtype).tiny * torch.finfo(y.dtype).eps
    assert np.all(np.abs(got - want) <= tol * np.abs(want) + tiny), np.abs(got - want).max()
    return y


@pytest.mark.parametrize("dtype", DTS)
@pytest.mark.parametrize("T,K", [(1, 1), (3, 7), (5, 16), (2, 1000), (64, 2048), (1, 4096), (3, 4097), (2, 20000)])
def test_quantize_rows(dtype, T, K):
    x = normal(T, K, seed=K, dtype=dtype)
    x[0, 0] = 0.5 * x[0].abs().max()          # a tie of the rounding
    c, s = quantize_rows(x)
    q, ws = ref64.quantise(np64(x))
    assert np.array_equal(np64(c), q)
    assert np.all(np.abs(np64(s) - ws[:, 0]) <= 2.0 ** -23 * ws[:, 0])


def test_quantize_special_rows():
    x = normal(9, 96, seed=1)
    x[0] = 0
    x[1, 3] = torch.inf
    x[2, 4] = torch.nan
    x[3] = torch.finfo(torch.float32).max
    x[4] *= 1e-38
    x[5] *= 1e-44                             # subnormal
    x[6, :] = -1.0
    x[7] *= 1e36
    c, s = quantize_rows(x)
    q, ws = ref64.quantise(np64(x[[0, 3, 4, 5, 6, 7, 8]]))
    assert np.array_equal(np64(c[[0, 3, 4, 5, 6, 7, 8]]), q)
    assert torch.isnan(s[1:3]).all() and (c[1:3] == 0).all()
    w = matrix(40, cols=96, seed=2)
    for rows in (x, x.repeat(3, 1)):
        y = int8_linear(rows, w)
        bad = torch.isnan(y).all(1)
        assert bad[1] and bad[2] and not torch.isnan(y[~bad]).any() and bad.sum() == 2 * (len(rows) // 9)
        assert (y[0] == 0).all()


def test_quantize_strides():
    base = normal(6, 101, seed=3, dtype=torch.bfloat16)
    for v in (base[:, 1:98], base[::2], base.t().contiguous().t(), base[:1].expand(3, -1), base.view(2, 3, 101)):
        c, s = quantize_rows(v)
        q, _ = ref64.quantise(np64(v))
        assert np.array_equal(np64(c), q) and s.shape == v.shape[:-1]
    assert quantize_rows(base[:0]).codes.shape == (0, 101)


@pytest.mark.parametrize("dtype", DTS)
@pytest.mark.parametrize("T", [1, 2, 3, 4, 5, 6, 7, 8, 9, 16, 17, 33, 100, 129, 300, 513])
@pytest.mark.parametrize("K,N", [(512, 256), (77, 33), (1000, 515)])
def test_linear(dtype, T, K, N):
    x = normal(T, K, seed=T, dtype=dtype)
    check_linear(x, matrix(N, cols=K, seed=N), torch.float32)


@pytest.mark.parametrize("T", [1, 3, 4, 5, 6])
def test_linear_few_rows_of_a_large_matrix(T):
    # above 16 M codes four rows and more run on the tensor cores
    w = matrix(8200, cols=2048, seed=2)
    x = normal(T, 2048, seed=T, dtype=torch.bfloat16)
    y = check_linear(x, w, torch.float32)
    assert torch.equal(int8_linear(torch.cat((x, x)), w, torch.float32), torch.cat((y, y)))


@pytest.mark.parametrize("T", [1, 8, 9, 70])
@pytest.mark.parametrize("K,N", [(1, 1), (16, 1), (15, 130), (4096, 64), (4111, 5), (30000, 17), (131072, 3)])
def test_linear_edges(T, K, N):
    x = normal(T, K, seed=T + K)
    w = matrix(N, cols=K, seed=N, pad=32)
    check_linear(x, w)
    for out in (torch.bfloat16, torch.float16):
        check_linear(x, w, out)


def test_linear_extremes_stay_exact():
    # every code at its limit: the largest sum 32 bits have to hold
    K = 131072
    for T in (1, 12):
        x = torch.ones(T, K, device="cuda")
        w = Int8Matrix(torch.full((20, K), 127, dtype=torch.int8, device="cuda"), torch.ones(20, device="cuda"))
        check_linear(x, w)
        w.codes.fill_(-128)
        y = int8_linear(x, w)
        assert torch.allclose(y, torch.full_like(y, -128.0 * K), rtol=1e-6)


def test_linear_strides_and_rows_beyond():
    base = normal(40, 130, seed=5, dtype=torch.bfloat16)
    w = matrix(96, cols=100, seed=6)
    for T in (4, 40):
        check_linear(base[:T, 1:101], w)
        check_linear(base[:T, ::1][:, 2:102], w)
    # a slice of a larger matrix
    big = matrix(300, cols=100, seed=7)
    check_linear(base[:20, :100], Int8Matrix(big.codes[64:200], big.scales[64:200]))
    check_linear(base[:3, :100], Int8Matrix(big.codes[64:200], big.scales[64:200]))
    assert int8_linear(base[:0, :100], w).shape == (0, 96)


def setup(E, I, H, T, k, dtype=torch.bfloat16, seed=0, absent=0.0):
    g = torch.Generator().manual_seed(seed)
    x = normal(T, H, seed=seed + 1, dtype=dtype)
    pop = -1.1 * torch.log(1.0 + torch.randperm(E, generator=g).float())
    top, ids = torch.topk(1.3 * torch.randn(T, E, generator=g) + pop, k, dim=1)
    w = torch.softmax(top, 1).cuda()
    ids = ids.int()
    if absent:
        ids[torch.rand(T, k, generator=g) < absent] = -1
    mats = [matrix(E, I, cols=H, seed=seed + 2), matrix(E, I, cols=H, seed=seed + 3), matrix(E, H, cols=I, seed=seed + 4)]
    return x, ids.cuda(), w, mats, normal(T, H, seed=seed + 5, dtype=dtype)


def check_experts(x, ids, w, mats, residual, rows=None):
    out = int8_experts(x, ids, w, *mats, residual=residual)
    torch.cuda.synchronize()
    pick = slice(None) if rows is None else rows
    m = [(np64(a.codes), np64(a.scales)) for a in mats]
    want = ref64.experts(np64(x[pick]), ids[pick].cpu().numpy(), np64(w[pick]), *m,
                         residual=None if residual is None else np64(residual[pick]))
    part = want - (0 if residual is None else np64(residual[pick]))
    got = np64(out[pick])
    norm = np.linalg.norm
    assert norm(got - want) <= 4e-3 * norm(part) + torch.finfo(x.dtype).eps / 2 * norm(want)
    return out


@pytest.mark.parametrize("dtype", DTS)
@pytest.mark.parametrize("E,I,H,T,k", [(16, 64, 128, 1, 2), (8, 256, 512, 3, 4), (24, 333, 712, 5, 3), (5, 40, 72, 40, 5),
                                       (64, 256, 512, 30, 4), (24, 360, 1000, 61, 3), (4, 96, 100, 300, 2),
                                       (16, 131, 257, 129, 3), (1, 32, 64, 700, 1), (3, 1, 1, 50, 2), (512, 64, 128, 41, 10)])
def test_experts(dtype, E, I, H, T, k):
    x, ids, w, mats, res = setup(E, I, H, T, k, dtype, seed=E + T)
    check_experts(x, ids, w, mats, res)
    assert check_error() == 0


@pytest.mark.parametrize("T", [2, 90])
def test_experts_absent_and_bad_ids(T):
    x, ids, w, mats, res = setup(16, 96, 256, T, 4, seed=3, absent=0.4)
    ids[0] = -1
    out = check_experts(x, ids, w, mats, res)
    assert torch.equal(out[0], res[0])
    out = check_experts(x, torch.full_like(ids, -1), w, mats, res)
    assert torch.equal(out, res)
    assert check_error() == 0
    none = int8_experts(x, torch.full_like(ids, -1), w, *mats)
    assert (none == 0).all()
    bad = ids.clone()
    bad[1, 0], bad[1, 1] = 16, -7
    check_experts(x, bad, w, mats, res)
    assert check_error() != 0 and check_error() == 0
    check_experts(x, ids, w, mats, None)


def test_experts_all_rows_on_one_expert_and_none_on_others():
    x, ids, w, mats, res = setup(32, 64, 128, 600, 3, seed=4)
    ids[:, 0], ids[:, 1], ids[:, 2] = 31, 7, 7      # the same expert twice in a row counts twice
    check_experts(x, ids, w, mats, res)


def test_experts_poison_stays_in_its_row():
    for T in (4, 80):
        x, ids, w, mats, res = setup(16, 96, 256, T, 4, seed=6)
        want = int8_experts(x, ids, w, *mats, residual=res)
        x[2, 5] = torch.nan
        x[3, 1] = torch.inf
        out = int8_experts(x, ids, w, *mats, residual=res)
        keep = [t for t in range(T) if t not in (2, 3)]
        assert torch.equal(out[keep], want[keep])
        assert torch.isnan(out[2:4]).all()


def test_experts_strides_residual_in_place_and_repeatable():
    for T in (3, 150):
        x, ids, w, mats, res = setup(16, 96, 256, T, 4, seed=7)
        want = int8_experts(x, ids, w, *mats, residual=res)
        wide = torch.zeros(T, 300, dtype=x.dtype, device="cuda")
        wide[:, 7:263] = x
        rw = torch.zeros(T, 259, dtype=x.dtype, device="cuda")
        rw[:, 1:257] = res
        assert torch.equal(int8_experts(wide[:, 7:263], ids, w, *mats, residual=rw[:, 1:257]), want)
        two = torch.cat((ids, ids), 1)
        assert torch.equal(int8_experts(x, two[:, :4], w, *mats, residual=res), want)
        for _ in range(5):
            assert torch.equal(int8_experts(x, ids, w, *mats, residual=res), want)


def test_rows_do_not_depend_on_their_batch():
    # every pair's product is the same whatever else is in the batch
    x, ids, w, mats, res = setup(16, 160, 256, 200, 4, seed=8)
    whole = int8_experts(x, ids, w, *mats, residual=res)
    assert torch.equal(int8_experts(x[50:150], ids[50:150], w[50:150], *mats, residual=res[50:150]), whole[50:150])
    y = int8_linear(x, matrix(300, cols=256, seed=9))
    assert torch.equal(int8_linear(x[100:120], matrix(300, cols=256, seed=9)), y[100:120])
    assert torch.equal(int8_linear(x[100:103], matrix(300, cols=256, seed=9)), y[100:103])


def test_two_streams_and_graphs():
    x, ids, w, mats, res = setup(16, 96, 256, 90, 4, seed=10)
    lin = matrix(500, cols=256, seed=11)
    want = int8_experts(x, ids, w, *mats, residual=res), int8_linear(x, lin)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        for s in streams:
            outs.append((int8_experts(x, ids, w, *mats, residual=res, stream=s), int8_linear(x, lin, stream=s)))
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o[0], want[0]) and torch.equal(o[1], want[1])
    buf, bids = x.clone(), ids.clone()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = int8_experts(buf, bids, w, *mats, residual=res), int8_linear(buf[:5], lin)
        graphs.append((g, out))
    x2, ids2 = setup(16, 96, 256, 90, 4, seed=20)[:2]
    buf.copy_(x2)
    bids.copy_(ids2)
    for g, _ in graphs:
        g.replay()
    torch.cuda.synchronize()
    ref = int8_experts(x2, ids2, w, *mats, residual=res), int8_linear(x2[:5], lin)
    for _, out in graphs:
        assert torch.equal(out[0], ref[0]) and torch.equal(out[1], ref[1])


@pytest.mark.parametrize("T", [1, 4])
def test_few_pairs_on_streams_and_in_graphs(T):
    # the two kernels of few pairs overlap (programmatic launch): back to back calls on changing inputs, on two
    # streams, and replays, with the routing made just before on the same stream
    from yanah_b200.routing import RouteRule, route_scored
    x, _, _, mats, res = setup(16, 96, 256, T, 4, seed=30)
    rule = RouteRule(4)

    def run(rows, logits):
        ids, w = route_scored(logits, rule)
        return int8_experts(rows, ids, w, *mats, residual=res)

    ins = [(normal(T, 256, seed=40 + i, dtype=x.dtype), normal(T, 16, seed=60 + i)) for i in range(12)]
    want = [run(*i) for i in ins]
    torch.cuda.synchronize()
    for i, w in zip(ins, want):
        ids, weights = route_scored(i[1], rule)
        m = [(np64(a.codes), np64(a.scales)) for a in mats]
        ref = ref64.experts(np64(i[0]), ids.cpu().numpy(), np64(weights), *m, residual=np64(res))
        assert np.linalg.norm(np64(w) - ref) <= (4e-3 + 2 ** -8) * np.linalg.norm(ref)
    for _ in range(3):
        assert all(torch.equal(run(*i), w) for i, w in zip(ins, want))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for n, i in enumerate(ins):
        with torch.cuda.stream(streams[n % 2]):
            got.append(run(*i))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    bx, bl = ins[0][0].clone(), ins[0][1].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        first = run(bx, bl)
        second = run(first, bl)
    for i, w in zip(ins, want):
        bx.copy_(i[0])
        bl.copy_(i[1])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(first, w) and torch.equal(second, run(w, i[1]))


def test_offsets_past_32_bits():
    # an output of more than 2^31 elements, and matrices of more than 2^31 bytes
    x = normal(14500, 32, seed=70, dtype=torch.bfloat16)
    w = matrix(151936, cols=32, seed=71)
    y = int8_linear(x, w)
    some = torch.tensor([0, 7000, 14499])
    want = ref64.linear(np64(x[some]), np64(w.codes[-500:]), np64(w.scales[-500:]))
    got = np64(y[some][:, -500:])
    assert np.all(np.abs(got - want) <= (2 ** -8 + 2 ** -21) * np.abs(want))
    del y
    E, I, H = 1024, 1088, 2048
    g = torch.Generator(device="cuda").manual_seed(72)
    codes = [torch.randint(-127, 128, s, generator=g, device="cuda", dtype=torch.int8) for s in ((E, I, H), (E, I, H), (E, H, I))]
    mats = [Int8Matrix(c, torch.full(c.shape[:2], 2e-4, device="cuda")) for c in codes]
    assert codes[0].numel() > 2 ** 31
    for T in (2, 60):
        x, res = normal(T, H, seed=73, dtype=torch.bfloat16), normal(T, H, seed=74, dtype=torch.bfloat16)
        ids = torch.full((T, 2), 1023, dtype=torch.int32, device="cuda")
        ids[:, 1] = 1000
        w = torch.full((T, 2), 0.5, device="cuda")
        out = int8_experts(x, ids, w, *mats, residual=res)
        m = [({1023: np64(a.codes[1023]), 1000: np64(a.codes[1000])}, np64(a.scales)) for a in mats]

        class At:   # the two experts that are used, by id
            shape = (E,)

            def __init__(self, d):
                self.d = d

            def __getitem__(self, e):
                return self.d[e]

        want = ref64.experts(np64(x[-2:]), ids[-2:].cpu().numpy(), np64(w[-2:]), *[(At(d), s) for d, s in m],
                             residual=np64(res[-2:]))
        got = np64(out[-2:])
        part = want - np64(res[-2:])
        assert np.linalg.norm(got - want) <= 4e-3 * np.linalg.norm(part) + 2 ** -8 * np.linalg.norm(want)


def test_refusals():
    x, ids, w, mats, res = setup(8, 64, 128, 4, 2, seed=12)
    lin = matrix(32, cols=128)
    with pytest.raises(ValueError):
        int8_linear(x[:, :100], lin)
    with pytest.raises(TypeError):
        int8_linear(x, Int8Matrix(lin.codes.float(), lin.scales))
    with pytest.raises(TypeError):
        int8_linear(x, lin, torch.float64)
    with pytest.raises(ValueError):
        int8_linear(x, mats[0])
    odd = torch.zeros(32, 130, dtype=torch.int8, device="cuda")[:, :128]
    with pytest.raises(_lib.YanahError):
        int8_linear(x, Int8Matrix(odd, lin.scales))
    with pytest.raises(TypeError):
        int8_experts(x, ids.long(), w, *mats)
    with pytest.raises(ValueError):
        int8_experts(x, ids, w[:, :1], *mats)
    with pytest.raises(_lib.YanahError):
        int8_experts(x, ids, w, mats[0], mats[1], mats[0])
    with pytest.raises(ValueError):
        int8_experts(x, ids, w, *mats, residual=res[:2])
    with pytest.raises(TypeError):
        int8_experts(x, ids, w, *mats, residual=res.float())
    with pytest.raises(RuntimeError):
        int8_linear(x.float().requires_grad_(), lin)
