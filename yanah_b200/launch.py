"""What the functional operators (``routing``, ``int8``, ``logprobs``) share: checks
of their tensor arguments, and running on a given stream or another device.

They allocate their outputs and workspaces with torch on the stream they run on, so
two calls never share memory, on one stream or on several, eager or captured. They
have no gradients: an argument that requires one is refused while gradients are on, and
so is one with a tangent (forward mode).
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

# element types of the C ABI (YN_F32, YN_BF16, YN_F16)
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


# A call of a few rows takes the host longer than the device: these checks ask a tensor for
# as little as they can (each attribute costs 0.1 to 0.3 us), and the operators allocate with
# sizes given one by one and with empty_like (1.3 us; with a tuple 1.8 us).
def check_floats(t: torch.Tensor, what: str) -> int:
    """A CUDA tensor of fp32, bf16 or fp16 without a gradient; returns the C ABI's code of its type."""
    code = DTYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"{what} must be float32, bfloat16 or float16, not {t.dtype}")
    if not t.is_cuda:
        raise ValueError(f"{what} must be a CUDA tensor")
    check_constant(t, what)
    return code


def check_constant(t: torch.Tensor, what: str) -> None:
    """A tensor that no derivative is asked of."""
    if t.requires_grad:
        check_no_grad(what)
    # only inside forward_ad.dual_level() has a tensor a tangent
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise RuntimeError(f"{what} has a tangent: this operator has no derivative")


def check_no_grad(what: str) -> None:
    """For an argument that requires a gradient."""
    if torch.is_grad_enabled():
        raise RuntimeError(f"{what} requires a gradient: this operator has none (call it under torch.no_grad())")


def check_like(t: torch.Tensor, index: int, shape: tuple, dtypes: tuple, what: str) -> None:
    """`t` on CUDA device `index`, of this shape and one of these types."""
    if t.shape != shape:
        raise ValueError(f"{what} must have shape {tuple(shape)}, not {tuple(t.shape)}")
    if t.dtype not in dtypes:
        raise TypeError(f"{what} must be {' or '.join(str(d) for d in dtypes)}, not {t.dtype}")
    if t.get_device() != index:
        raise ValueError(f"{what} is on {t.device}, not on cuda:{index}")
    check_constant(t, what)


def rows_of(t: torch.Tensor, what: str) -> Tuple[torch.Tensor, int, int, int]:
    """`t` as rows whose elements are adjacent and which do not overlap (copied where it is laid out otherwise),
    their number, length and stride."""
    if t.dim() != 2:
        raise ValueError(f"{what} must have two dimensions, not {t.dim()}")
    n, c = t.shape
    s0, s1 = t.stride()
    if (c > 1 and s1 != 1) or (n > 1 and s0 < c):
        return t.contiguous(), n, c, c
    return t, n, c, s0 if n > 1 else c


def raw_stream(index: int) -> int:
    """The current stream of CUDA device `index` as the C ABI takes it."""
    return torch._C._cuda_getCurrentRawStream(index)


def elsewhere(index: int, stream: Optional[torch.cuda.Stream]) -> bool:
    """Whether a call has to leave the current device or stream."""
    return stream is not None or index != torch._C._cuda_getDevice()


def run_there(fn, device: torch.device, stream: Optional[torch.cuda.Stream], tensors):
    """fn() with `device` and `stream` (None: the device's current one) current. The caching allocator is told that
    the tensors are in use on a stream that was given."""
    if stream is not None and stream.device != device:
        raise ValueError(f"the stream is on {stream.device}, the tensors on {device}")
    with torch.cuda.device(device):
        if stream is None:
            return fn()
        with torch.cuda.stream(stream):
            for t in tensors:
                if t is not None and t.is_cuda:   # fn refuses others
                    t.record_stream(stream)
            return fn()
