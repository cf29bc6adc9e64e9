"""What the functional operators (``routing``, ``int8``, ``logprobs``) share: checks
of their tensor arguments, and running on a given stream or another device.

They allocate their outputs and workspaces with torch on the stream they run on, so
two calls never share memory, on one stream or on several, eager or captured. They
have no gradients: an argument that requires one is refused while gradients are on.
"""
from __future__ import annotations

from typing import Optional

import torch

# element types of the C ABI (YN_F32, YN_BF16, YN_F16)
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def check_floats(t: torch.Tensor, what: str) -> None:
    """A CUDA tensor of fp32, bf16 or fp16 without a gradient."""
    if t.dtype not in DTYPES:
        raise TypeError(f"{what} must be float32, bfloat16 or float16, not {t.dtype}")
    if not t.is_cuda:
        raise ValueError(f"{what} must be a CUDA tensor")
    if t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{what} requires a gradient: this operator has none (call it under torch.no_grad())")


def check_like(t: torch.Tensor, like: torch.Tensor, shape: tuple, dtypes: tuple, what: str) -> None:
    """`t` on the device of `like`, of this shape and one of these types."""
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what} must have shape {tuple(shape)}, not {tuple(t.shape)}")
    if t.dtype not in dtypes:
        raise TypeError(f"{what} must be {' or '.join(str(d) for d in dtypes)}, not {t.dtype}")
    if t.device != like.device:
        raise ValueError(f"{what} is on {t.device}, not on {like.device}")


def rows_of(t: torch.Tensor, what: str) -> torch.Tensor:
    """`t` as rows whose elements are adjacent and which do not overlap; copied where it is laid out otherwise."""
    if t.dim() != 2:
        raise ValueError(f"{what} must have two dimensions, not {t.dim()}")
    n, c = t.shape
    if (c > 1 and t.stride(1) != 1) or (n > 1 and t.stride(0) < c):
        return t.contiguous()
    return t


def row_stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])


def raw_stream(device: torch.device) -> int:
    """The current stream of a device as the C ABI takes it."""
    return torch._C._cuda_getCurrentRawStream(device.index)


def elsewhere(device: torch.device, stream: Optional[torch.cuda.Stream]) -> bool:
    """Whether a call has to leave the current device or stream."""
    return stream is not None or device.index != torch.cuda.current_device()


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
                if t is not None:
                    t.record_stream(stream)
            return fn()
