"""What the token-generation entry points share: tensors of heads, streams and devices.

Rows of heads are CUDA tensors [tokens, heads, width] in float32, bfloat16 or float16 with any
token and head strides and a unit stride along the width, so that a slice of a projection's output
is taken as it lies.
"""

from __future__ import annotations

import contextlib

import torch

from tgcb import _lib
from tgcb.errors import ConfigError

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}

_here = contextlib.nullcontext()


def check_rows(name: str, t: torch.Tensor, like: torch.Tensor | None = None) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dim() != 3 or t.dtype not in DTYPES:
        raise ConfigError(f"{name} must be a CUDA tensor [tokens, heads, width] in float32, bfloat16 or float16")
    if t.stride(2) != 1 and t.shape[2] != 1:
        raise ConfigError(f"{name} must have a unit stride along its width")
    if like is not None and (t.dtype != like.dtype or t.device != like.device):
        raise ConfigError(f"{name} must have the type and device of the other rows")


def check_vector(name: str, t: torch.Tensor, length: int, dtypes: tuple, device: torch.device) -> None:
    if not isinstance(t, torch.Tensor) or t.device != device or t.dtype not in dtypes:
        raise ConfigError(f"{name} must be a tensor on {device} in {' or '.join(str(d) for d in dtypes)}")
    if t.dim() != 1 or t.shape[0] != length or (length > 1 and t.stride(0) != 1):
        raise ConfigError(f"{name} must be a contiguous vector of {length}, got {tuple(t.shape)}")


def check_written(name: str, t: torch.Tensor) -> None:
    """Refuse an output in which two elements share memory."""
    span = t.shape[2]
    for size, stride in sorted(((t.shape[0], t.stride(0)), (t.shape[1], t.stride(1))), key=lambda x: x[1]):
        if size > 1:
            if stride < span:
                raise ConfigError(f"{name} must not overlap itself")
            span += (size - 1) * stride


def _reach(t: torch.Tensor) -> tuple[int, int]:
    first = t.data_ptr()
    return first, first + (sum((n - 1) * s for n, s in zip(t.shape, t.stride(), strict=True)) + 1) * t.element_size()


def overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors of rows may share memory. Slices of the same wider rows, side by side, do not."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    (a0, a1), (b0, b1) = _reach(a), _reach(b)
    if a1 <= b0 or b1 <= a0:
        return False
    for dim in (0, 1):  # both repeat with one stride, within which each has its own part
        step = a.stride(dim) * a.element_size()
        if a.dtype == b.dtype and a.shape[dim] == b.shape[dim] and a.stride(dim) == b.stride(dim):
            a_end, b_end = _reach(a.narrow(dim, 0, 1))[1], _reach(b.narrow(dim, 0, 1))[1]
            if max(a_end, b_end) - min(a0, b0) <= step:
                return not (a_end <= b0 or b_end <= a0)
    return True


def check_apart(name: str, out: torch.Tensor, other_name: str, other: torch.Tensor, *, same_allowed: bool = False) -> None:
    if same_allowed and out.data_ptr() == other.data_ptr() and out.shape == other.shape and out.stride() == other.stride():
        return
    if overlap(out, other):
        raise ConfigError(f"{name} overlaps {other_name}")


def rows(t: torch.Tensor) -> _lib.Heads:
    return _lib.Heads(t.data_ptr(), t.stride(0), t.stride(1))


def on_device(device: torch.device):
    """A context in which `device` is current, and set up."""
    index = device.index
    _lib.ensure_device(index)
    return _here if torch.cuda.current_device() == index else torch.cuda.device(index)


def on_stream(device: torch.device, stream):
    """A context in which `stream` (None: the current one) is current, for what a call allocates."""
    if stream is None:
        return _here
    if stream.device != device:
        raise ConfigError(f"the stream is on {stream.device}, the tensors on {device}")
    return torch.cuda.stream(stream)


def raw(device: torch.device, stream) -> int:
    return (stream if stream is not None else torch.cuda.current_stream(device)).cuda_stream
