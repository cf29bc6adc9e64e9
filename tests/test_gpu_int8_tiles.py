"""GPU tests of the 8-bit tensor-core product's tile shapes: tiles cut even over the pairs of SMs
(few rows of more than 256 channels per pair: 18944 on 148 SMs), whose boxes have any even height up
to 128, and gate and up matrices that lie in memory in either order, alike or not.

Bounds: those of the linear and the experts' tests.
"""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from tests import ref64
from tests.test_gpu_int8 import DTS, check_experts, matrix, normal, np64, setup
from yanah_b200 import _lib
from yanah_b200.int8 import Int8Matrix, int8_experts, int8_linear

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N,K", [(18944, 48), (18945, 200), (18949, 48), (20000, 1000), (37888, 200), (37889, 48),
                                 (50257, 200), (100003, 48), (100003, 200)])
def test_even_tiles(N, K):
    w = matrix(N, cols=K, seed=N)
    codes, scales = np64(w.codes), np64(w.scales)
    for T in (4, 6, 17, 32):        # four rows are made by dp4a where the matrix is small
        x = normal(T, K, seed=T, dtype=DTS[T % 3])
        want = ref64.linear(np64(x), codes, scales)
        for out in DTS:
            y = int8_linear(x, w, out)
            got = np64(y)
            tol = torch.finfo(out).eps / 2 + 2.0 ** -21
            tiny = torch.finfo(out).tiny * torch.finfo(out).eps
            assert np.all(np.abs(got - want) <= tol * np.abs(want) + tiny), (T, out)
        # the same rows among more than 32, in tiles of 128 channels a block
        more = int8_linear(x.repeat(10, 1)[:T + 33], w, out)
        assert torch.equal(more[:T], y)


def test_even_tiles_write_their_rows_and_channels_only():
    T, K, N = 6, 96, 20001
    w, x = matrix(N, cols=K, seed=3), normal(T, K, seed=4)
    want = int8_linear(x, w)
    lib = _lib.lib()
    nb = lib.yn_i8_linear_ws_bytes(T, K)
    ws = torch.empty(nb, dtype=torch.uint8, device="cuda")
    m = _lib.I8Mat(w.codes.data_ptr(), w.scales.data_ptr(), w.codes.stride(0), 0, 0, 1, N, K)
    for code, dtype in ((0, torch.float32), (1, torch.bfloat16), (2, torch.float16)):
        for first, pitch in ((8, N + 21), (7, N + 22), (6, N + 24)):
            buf = torch.full((T + 2, pitch), 7.0, dtype=dtype, device="cuda")
            y = buf[1:1 + T, first:first + N]
            _lib.check(lib.yn_i8_linear(C.byref(m), x.data_ptr(), 0, K, T, y.data_ptr(), code, pitch, ws.data_ptr(), nb,
                                        torch.cuda.current_stream().cuda_stream))
            torch.cuda.synchronize()
            assert torch.equal(y, want.to(dtype))
            y.fill_(7.0)
            assert (buf == 7.0).all()


@pytest.mark.parametrize("dtype", DTS[:2])
@pytest.mark.parametrize("I,H,T,k", [(64, 128, 90, 2), (160, 256, 40, 4), (160, 256, 700, 3), (131, 200, 90, 2)])
def test_gate_and_up_in_either_order(I, H, T, k, dtype):
    E = 6
    x, ids, w, (gate, up, down), res = setup(E, I, H, T, k, dtype, seed=50)
    want = check_experts(x, ids, w, (gate, up, down), res)
    st = gate.codes.stride(1)

    def place(dim, order):
        """gate and up as slices of one buffer, side by side along `dim`."""
        shape = [E, I, st]
        shape.insert(dim, 2)
        codes = torch.zeros(shape, dtype=torch.int8, device="cuda")
        out = []
        for i, m in zip(order, (gate, up)):
            c = codes.select(dim, i)
            c[..., :H] = m.codes
            out.append(Int8Matrix(c[..., :H], m.scales))
        return out

    for dim in (0, 1, 2):
        for order in ((0, 1), (1, 0)):
            g, u = place(dim, order)
            assert (g.codes.data_ptr() < u.codes.data_ptr()) == (order == (0, 1))
            assert torch.equal(int8_experts(x, ids, w, g, u, down, residual=res), want), (dim, order)
    # not alike: rows of another pitch
    wide = torch.zeros(E, I, st + 16, dtype=torch.int8, device="cuda")
    wide[..., :H] = up.codes
    assert torch.equal(int8_experts(x, ids, w, gate, Int8Matrix(wide[..., :H], up.scales), down, residual=res), want)
    assert torch.equal(int8_experts(x, ids, w, Int8Matrix(wide[..., :H], up.scales), up, down, residual=res),
                       int8_experts(x, ids, w, up, up, down, residual=res))


@pytest.mark.parametrize("dtype", DTS)
@pytest.mark.parametrize("k,rows", [(1, (119, 120, 121)), (2, (59, 60, 61)), (3, (39, 40, 41))])
def test_chunks_of_either_size(k, rows, dtype):
    # 3 experts: up to 120 pairs are cut into chunks of 64 rows, more into chunks of 256
    x, ids, w, mats, res = setup(3, 100, 136, 200, k, dtype, seed=60 + k)
    whole = check_experts(x, ids, w, mats, res)
    for n in rows:
        assert torch.equal(int8_experts(x[:n], ids[:n], w[:n], *mats, residual=res[:n]), whole[:n])


def at_the_end(t):
    """A copy of a matrix's codes that ends where its memory does (a block of its own of whole 2 MiB pages)."""
    E, N, K = t.shape
    pitch = (K + 15) // 16 * 16
    size = E * N * pitch
    block = torch.zeros((size + (20 << 20) + (2 << 20) - 1) >> 21 << 21, dtype=torch.int8, device="cuda")
    out = block[block.numel() - size:].view(E, N, pitch)
    out[..., :K] = t
    return out[..., :K]


@pytest.mark.parametrize("E,I,H,T,k", [(9, 32, 2, 149, 7), (3, 16, 100, 60, 2), (2, 64, 128, 40, 2), (5, 80, 255, 30, 4),
                                       (4, 131, 300, 90, 1), (1, 208, 374, 10, 8)])
def test_matrices_at_the_end_of_their_memory(E, I, H, T, k):
    # tiles that lie partly or wholly past the last rows: nothing there is touched
    x, ids, w, mats, res = setup(max(E, k), I, H, T, k, seed=70 + E)
    mats = [Int8Matrix(m.codes[:E], m.scales[:E]) for m in mats]
    ids = ids % E
    want = check_experts(x, ids, w, mats, res)
    for which in ((0,), (1,), (2,), (0, 1, 2), (1, 0, 2)):
        moved = list(mats)
        for i in which:
            moved[i] = Int8Matrix(at_the_end(mats[i].codes), mats[i].scales)
        assert torch.equal(int8_experts(x, ids, w, *moved, residual=res), want), which
    for i in range(3):      # a product's matrix
        one = Int8Matrix(at_the_end(mats[i].codes[:1])[0], mats[i].scales[0])
        rows = normal(40, one.codes.shape[1], seed=i)
        assert torch.equal(int8_linear(rows, one), int8_linear(rows, Int8Matrix(mats[i].codes[0], mats[i].scales[0])))


@pytest.mark.parametrize("T", [3, 90])
def test_matrices_interleaved_row_by_row(T):
    E, I, H, k = 6, 100, 200, 4
    x, ids, w, mats, res = setup(E, I, H, T, k, seed=80)
    want = check_experts(x, ids, w, mats, res)

    def interleaved(m, extra=0):
        n, _, c = m.codes.shape
        buf = torch.zeros(m.codes.shape[1], n + extra, (c + 15) // 16 * 16, dtype=torch.int8, device="cuda")
        v = buf[:, :n, :c].transpose(0, 1)
        v.copy_(m.codes)
        return Int8Matrix(v, m.scales)

    for extra in (0, 2):
        inter = [interleaved(m, extra) for m in mats]
        for pick in ((1, 1, 1), (1, 0, 0), (0, 1, 0), (0, 0, 1)):
            got = int8_experts(x, ids, w, *[inter[i] if p else mats[i] for i, p in enumerate(pick)], residual=res)
            assert torch.equal(got, want), (extra, pick)


def test_one_row_matrices_of_any_distance():
    x, ids, w, (gate, up, down), res = setup(5, 1, 40, 90, 2, seed=81)
    want = check_experts(x, ids, w, (gate, up, down), res)
    wide = torch.zeros(5, 3, 80, dtype=torch.int8, device="cuda")
    wide[:, 1, :40] = gate.codes[:, 0]
    assert torch.equal(int8_experts(x, ids, w, Int8Matrix(wide[:, 1:2, :40], gate.scales), up, down, residual=res), want)
