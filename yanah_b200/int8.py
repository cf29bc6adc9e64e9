"""Matrix products in 8-bit integers with one scale per row (token) and one per output
channel, and the routed experts of an MoE layer in that form.

Beside the group-affine products of the records (``yn_qlinear``, ``yn_tc_experts``):
those keep the checkpoint's 2 / 4 / 8-bit codes, these trade memory (one byte per
weight) for the tensor cores' integer rate. ``PrefillStack(experts="int8")`` runs its
prompt passes on them, ``speculation.verify_rows`` its LM head.

    w = quantize_rows(weight)                  # (N, K) -> codes, channel scales; once
    y = int8_linear(x, w)                      # (T, K) -> (T, N)
    out = int8_experts(x, ids, weights, gate, up, down, residual=h)

Every call quantises the rows it is given (code = the whole number nearest to
127 x / max|x|). Sums are exact in 32 bits.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

import torch

from . import _lib
from .launch import DTYPES, check_constant, check_floats, check_like, elsewhere, raw_stream, rows_of, run_there


class Int8Matrix(NamedTuple):
    """``codes`` (N, K) int8, or (E, N, K) for a matrix per expert, and ``scales`` (N) or
    (E, N) fp32 of the output channels. Rows of codes start at multiples of 16 bytes, as
    ``quantize_rows`` lays them out; matrices lie whole rows apart, or are interleaved row by
    row."""
    codes: torch.Tensor
    scales: torch.Tensor


def quantize_rows(x: torch.Tensor, stream: Optional[torch.cuda.Stream] = None) -> Int8Matrix:
    """Rows (..., K) as 8-bit codes with one scale each: activations per token, weights
    per output channel. A row with an infinity or a NaN gets a NaN scale."""
    dtype, dev = check_floats(x, "x"), x.get_device()
    if elsewhere(dev, stream):
        return run_there(lambda: quantize_rows(x), x.device, stream, (x,))
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("x must have at least one column")
    lead, k = x.shape[:-1], x.shape[-1]
    flat, rows, k, stride = rows_of(x.reshape(-1, k), "x")
    pitch = (k + 15) // 16 * 16
    codes = x.new_empty(rows, pitch, dtype=torch.int8)
    scales = x.new_empty(rows, dtype=torch.float32)
    _lib.check(_lib.lib().yn_i8_quant_rows(flat.data_ptr(), dtype, stride, rows, k, codes.data_ptr(), pitch,
                                           scales.data_ptr(), raw_stream(dev)))
    return Int8Matrix(codes.view(*lead, pitch)[..., :k], scales.view(lead))


def _mat(w: Int8Matrix, index: int, what: str) -> _lib.I8Mat:
    codes, scales = w
    shape, strides, s_strides = codes.shape, codes.stride(), scales.stride()
    if codes.dtype is not torch.int8 or scales.dtype is not torch.float32:
        raise TypeError(f"{what} must have int8 codes and float32 scales")
    if len(shape) == 3:
        mats, n, k = shape
        alike = scales.shape == (mats, n)
    elif len(shape) == 2:
        mats, (n, k) = 1, shape
        alike = scales.shape == (n,)
    else:
        alike = False
    if not alike:
        raise ValueError(f"{what}: codes (N, K) or (E, N, K) with scales (N) or (E, N)")
    if codes.get_device() != index or scales.get_device() != index:
        raise ValueError(f"{what} is not on cuda:{index}")
    check_constant(scales, f"{what}'s scales")
    if (k > 1 and strides[-1] != 1) or (n > 1 and s_strides[-1] != 1):
        raise ValueError(f"{what}: a row's codes and a matrix's scales must be adjacent")
    rs = strides[-2] if n > 1 else (k + 15) // 16 * 16
    if mats > 1:
        return _lib.I8Mat(codes.data_ptr(), scales.data_ptr(), rs, strides[0], s_strides[0], mats, n, k)
    return _lib.I8Mat(codes.data_ptr(), scales.data_ptr(), rs, rs * n, n, mats, n, k)


def int8_linear(x: torch.Tensor, w: Int8Matrix, out_dtype: Optional[torch.dtype] = None,
                stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """x (T, K) in fp32, bf16 or fp16 times the transpose of w (N, K): (T, N) in
    ``out_dtype`` (default: that of x), rounded once from fp32: the sum times the row's
    scale, times the channel's. Any number of rows. ``check_error`` reports a product that
    did not finish."""
    dtype, dev = check_floats(x, "x"), x.get_device()
    if elsewhere(dev, stream):
        return run_there(lambda: int8_linear(x, w, out_dtype), x.device, stream, (x, *w))
    x, rows, k, stride = rows_of(x, "x")
    if w.codes.dim() != 2:
        raise ValueError("w must be one matrix (N, K)")
    m = _mat(w, dev, "w")
    if k != m.cols:
        raise ValueError(f"x has {k} columns, w {m.cols}")
    out_dtype = out_dtype or x.dtype
    if out_dtype not in DTYPES:
        raise TypeError(f"out_dtype must be float32, bfloat16 or float16, not {out_dtype}")
    n = m.rows
    y = x.new_empty(rows, n, dtype=out_dtype)
    lib = _lib.lib()
    nb = lib.yn_i8_linear_ws_bytes(rows, k)
    ws = x.new_empty(nb, dtype=torch.uint8) if nb else None
    _lib.check(lib.yn_i8_linear(C.byref(m), x.data_ptr(), dtype, stride, rows, y.data_ptr(), DTYPES[out_dtype], n,
                                None if ws is None else ws.data_ptr(), nb, raw_stream(dev)))
    return y


def int8_experts(x: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor, gate: Int8Matrix, up: Int8Matrix,
                 down: Int8Matrix, residual: Optional[torch.Tensor] = None,
                 stream: Optional[torch.cuda.Stream] = None, out: Optional[torch.Tensor] = None,
                 err: Optional[torch.Tensor] = None) -> torch.Tensor:
    """residual + sum over a row's experts of weight * down(silu(gate x) * up x).

    x (T, H); ids (T, k) int32 and weights (T, k) fp32 as ``routing.route_scored``
    returns them: an id of -1 has no expert (any other id outside [0, E) is left out and
    reported by ``check_error``, or in ``err``, (1) int32, an error word of the caller's own).
    gate, up: (E, I, H); down: (E, H, I). The activations are quantised per (row, expert),
    the sum is fp32 and rounded once to the type of x.
    ``out``: (T, H) to write, rows of adjacent elements; it may be the residual."""
    dtype, dev = check_floats(x, "x"), x.get_device()
    if elsewhere(dev, stream):
        return run_there(lambda: int8_experts(x, ids, weights, gate, up, down, residual, out=out, err=err), x.device,
                         stream, (x, ids, weights, residual, out, err, *gate, *up, *down))
    x, rows, h, stride = rows_of(x, "x")
    if ids.dim() != 2:
        raise ValueError("ids must be (T, k)")
    k = ids.shape[1]
    check_like(ids, dev, (rows, k), (torch.int32,), "ids")
    check_like(weights, dev, (rows, k), (torch.float32,), "weights")
    g, u, d = _mat(gate, dev, "gate"), _mat(up, dev, "up"), _mat(down, dev, "down")
    if g.cols != h:
        raise ValueError(f"x has {h} columns, gate {g.cols}")
    ids, weights = ids.contiguous(), weights.contiguous()
    p_res, res_stride, out_stride = None, 0, h
    if residual is not None:
        check_like(residual, dev, (rows, h), (x.dtype,), "residual")
        residual, _, _, res_stride = rows_of(residual, "residual")
        p_res = residual.data_ptr()
    if out is None:
        out = x.new_empty(rows, h)
    else:
        check_like(out, dev, (rows, h), (x.dtype,), "out")
        same, _, _, out_stride = rows_of(out, "out")
        if same is not out:
            raise ValueError("out must have rows of adjacent elements that do not overlap")
    if err is not None:
        check_like(err, dev, (1,), (torch.int32,), "err")
    lib = _lib.lib()
    nb = lib.yn_i8_experts_ws_bytes(rows, k, g.n_mats, h, g.rows, dtype)
    ws = x.new_empty(nb, dtype=torch.uint8)
    _lib.check(lib.yn_i8_experts_err(C.byref(g), C.byref(u), C.byref(d), x.data_ptr(), dtype, stride, rows,
                                     ids.data_ptr(), weights.data_ptr(), k, p_res, res_stride, out.data_ptr(), out_stride,
                                     ws.data_ptr(), nb, None if err is None else err.data_ptr(), raw_stream(dev)))
    return out


def check_error(device=None) -> int:
    """Read and clear the error word of the 8-bit products on a device (synchronises its
    current stream): 0, or a code as ``CudaMoEBackend.check_error`` returns, of an id outside
    the experts or a wait inside a product that ran out (1 s: that call's output is wrong). All
    calls on the device share the word, but for those of ``int8_experts`` with one of their own."""
    code = C.c_int32(0)
    with torch.cuda.device(device):
        _lib.check(_lib.lib().yn_i8_error(torch.cuda.current_stream().cuda_stream, C.byref(code)))
    return code.value
