"""GPU tests of the token log probabilities against a plain 64-bit implementation.

Ids and ranks are compared for equality. fp32 results: log S = log1p(R) where R is a
sum of ex2 approximations, each within 2^-22 of itself plus the rounding of its
exponent (|y| 2^-24 for an exponent y = (z - m) log2 e, weighted by 2^y: below 2^-23),
so R and the entropy's sum are within 2^-20 of themselves with their summation error;
a log probability adds one rounding of z - m and one of the result. 2e-6 of
(1 + |value|) is asked, and where the token is the row's maximum and holds nearly all
the mass 4e-6 of the value itself.
"""
from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from tests import ref64
from yanah_b200.logprobs import token_logprobs

pytestmark = pytest.mark.gpu


def check(z, tokens, n):
    r = token_logprobs(z, tokens, n_top=n)
    torch.cuda.synchronize()
    want = ref64.logprobs(z.float().cpu().numpy(), tokens.cpu().numpy(), n)
    assert np.array_equal(r.rank.cpu().numpy(), want["rank"])
    close(r.logprob, want["logprob"])
    close(r.entropy, want["entropy"])
    if n:
        assert np.array_equal(r.top_ids.cpu().numpy(), want["top_ids"])
        close(r.top_logprobs, want["top_logprobs"])
    return r


def close(got, want):
    got = got.cpu().numpy().astype(np.float64)
    fin = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[~fin], want[~fin], equal_nan=True)
    err = np.abs(got[fin] - want[fin])
    assert np.all(err <= 2e-6 * (1 + np.abs(want[fin]))), err.max()


def logits(T, V, dtype=torch.float32, seed=0, std=3.0):
    g = torch.Generator().manual_seed(seed)
    z = std * torch.randn(T, V, generator=g)
    z[:, :: max(1, V // 7)] += 9
    tokens = torch.randint(0, V, (T,), generator=g)
    tokens[::2] = z[::2].argmax(1)
    return z.to(dtype).cuda(), tokens.int().cuda()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,V,n", [(1, 1, 1), (3, 2, 2), (1, 151936, 20), (5, 100003, 5), (2, 257, 64), (7, 4096, 1),
                                   (330, 33, 0), (300, 9001, 8), (300, 70001, 20), (4, 65536, 0)])
def test_shapes(dtype, T, V, n):
    check(*logits(T, V, dtype, seed=V), n)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T", [6, 300])
def test_masks_and_special_rows(dtype, T):
    V = 20011
    z, tokens = logits(T, V, dtype, seed=2)
    low = torch.finfo(dtype).min
    z[0] = -torch.inf                       # nothing to answer with
    z[1, 3:] = -torch.inf                   # fewer than n left
    tokens[1] = 7
    z[2, 11] = torch.inf
    z[2, 4000] = torch.inf
    tokens[2] = 4000
    z[3, V - 1] = torch.nan
    z[4] = low
    z[5, 1000:] = low
    tokens[5] = 1500
    check(z, tokens, 8)
    check(z, torch.full_like(tokens, -1), 3)
    tokens[:] = V
    check(z, tokens, 0)
    m = torch.rand(V, generator=torch.Generator().manual_seed(3)) < 0.97
    z[:, m.cuda()] = -torch.inf
    check(z, logits(T, V, dtype, seed=2)[1], 20)


@pytest.mark.parametrize("T", [2, 300])
def test_ties_come_by_id(T):
    # rows where far more elements share a value than the candidate buffer holds
    V = 30000
    z = torch.zeros(T, V, device="cuda")
    z[1::2] = (torch.arange(V, device="cuda") % 3).float()
    tokens = torch.full((T,), 17, dtype=torch.int32, device="cuda")
    tokens[-1] = V - 1
    check(z, tokens, 33)
    check(z.bfloat16(), tokens, 33)
    # equal values around block and vector borders
    z = torch.full((T, V), -5.0, device="cuda")
    z[:, [7, 8, 2047, 2048, 8191, 8192, V - 1]] = 2.0
    check(z, tokens, 10)


def test_one_token_has_nearly_all_mass():
    # log S far below one ulp of one: the relative accuracy of the log probability must stay
    for margin in (10.0, 30.0, 60.0):
        for V in (300, 50000):
            z = torch.full((3, V), -3.0, device="cuda")
            z[:, V // 2] = margin
            tokens = torch.full((3,), V // 2, dtype=torch.int32, device="cuda")
            r = token_logprobs(z, tokens, n_top=1)
            want = ref64.logprobs(z.cpu().numpy(), tokens.cpu().numpy(), 1)
            assert np.allclose(r.logprob.cpu().numpy(), want["logprob"], rtol=4e-6, atol=1e-44)
            assert np.allclose(r.top_logprobs.cpu().numpy(), want["top_logprobs"], rtol=4e-6, atol=1e-44)
            assert np.allclose(r.entropy.cpu().numpy(), want["entropy"], rtol=1e-5, atol=1e-44)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_alignment(dtype):
    base, _ = logits(9, 5003, dtype, seed=4)
    tok = torch.arange(9, dtype=torch.int32, device="cuda") * 100
    check(base[:, 1:4001], tok, 5)
    check(base[:, 5:1004], tok, 5)
    check(base[::3, 3:], tok[:3], 5)
    check(base.t().contiguous().t(), tok, 5)
    # what lies beside a row in the same 16 bytes must not reach it
    whole, _ = logits(4, 1003, dtype, seed=5)
    # (not compared with a copy of the row bit by bit: which thread sums an element depends on
    # where the row lies inside its 16 bytes)
    whole[:, :3] = torch.nan
    whole[:, 1000:] = torch.inf
    check(whole[:, 3:1000], tok[:4], 4)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T", [2, 300])
def test_signed_zeros_are_equal_and_denormals_are_not(dtype, T):
    V = 5000
    z = torch.full((T, V), -1.0, dtype=dtype, device="cuda")
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps       # the smallest value of the type
    z[:, 100] = -0.0
    z[:, 3000] = 0.0
    z[:, 3001] = -tiny
    z[:, 4999] = tiny
    z[1::2, 4999] = -2 * tiny
    for t in (100, 3000, 3001, 4999):
        check(z, torch.full((T,), t, dtype=torch.int32, device="cuda"), 6)


def test_large_offsets():
    # element offsets past 2^31
    V, T = 151936, 14200
    z = torch.zeros(T, V, dtype=torch.bfloat16, device="cuda")
    z[T - 1] = logits(1, V, torch.bfloat16, seed=6)[0][0]
    tok = torch.full((T,), 5, dtype=torch.int32, device="cuda")
    r = token_logprobs(z, tok, n_top=4)
    want = ref64.logprobs(z[T - 1:].float().cpu().numpy(), [5], 4)
    assert r.rank[T - 1].item() == want["rank"][0]
    assert np.array_equal(r.top_ids[T - 1].cpu().numpy(), want["top_ids"][0])
    assert r.top_ids[0].tolist() == [0, 1, 2, 3]


def test_streams_graphs_and_no_tokens():
    z, tokens = logits(5, 50001, seed=8)
    want = token_logprobs(z, tokens, n_top=6)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = token_logprobs(z, tokens, n_top=6, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    buf = z.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = token_logprobs(buf, tokens, n_top=6)
    for seed in (9, 10):
        new = logits(5, 50001, seed=seed)[0]
        buf.copy_(new)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(token_logprobs(new, tokens, n_top=6), out))
    r = token_logprobs(z)
    assert r.logprob is None and r.rank is None and r.top_ids is None
    assert torch.equal(r.entropy, want.entropy)
    assert token_logprobs(z[:0], tokens[:0], n_top=3).top_ids.shape == (0, 3)


def test_refusals():
    z, tokens = logits(2, 64)
    for bad in (dict(n_top=65), dict(n_top=-1), dict(tokens=tokens[:1])):
        with pytest.raises(ValueError):
            token_logprobs(z, bad.get("tokens", tokens), n_top=bad.get("n_top", 0))
    with pytest.raises(TypeError):
        token_logprobs(z, tokens.long())
    with pytest.raises(TypeError):
        token_logprobs(z.double(), tokens)
    with pytest.raises(ValueError):
        token_logprobs(z[0], tokens)
