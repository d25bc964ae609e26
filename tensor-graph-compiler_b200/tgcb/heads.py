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
    if t.stride()[2] != 1 and t.shape[2] != 1:
        raise ConfigError(f"{name} must have a unit stride along its width")
    if like is not None and (t.dtype is not like.dtype or t.get_device() != like.get_device()):
        raise ConfigError(f"{name} must have the type and device of the other rows")


def check_vector(name: str, t: torch.Tensor, length: int, dtypes: tuple, index: int) -> None:
    """A contiguous vector on CUDA device ``index``."""
    if not isinstance(t, torch.Tensor) or t.get_device() != index or t.dtype not in dtypes:
        raise ConfigError(f"{name} must be a tensor on cuda:{index} in {' or '.join(str(d) for d in dtypes)}")
    if t.shape != (length,) or not t.is_contiguous():
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
    """Whether two tensors of rows may share memory. Slices of the same wider rows, side by side, do not, nor do parts of each head."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    (a0, a1), (b0, b1) = _reach(a), _reach(b)
    if a1 <= b0 or b1 <= a0:
        return False
    if a.dtype != b.dtype:
        return True
    # Where both repeat with one stride, within which one step of each has its place, only equal steps can meet: on to one step of
    # both, from the larger of the two strides to the smaller.
    for dim in sorted((0, 1), key=a.stride, reverse=True):
        if a.shape[dim] == b.shape[dim] == 1:
            continue
        if min(a.shape[dim], b.shape[dim]) == 1 or a.stride(dim) != b.stride(dim):
            return True
        step = a.stride(dim) * a.element_size()
        a, b = a.narrow(dim, 0, 1), b.narrow(dim, 0, 1)
        a1, b1 = _reach(a)[1], _reach(b)[1]
        if max(a1, b1) - min(a0, b0) > step:
            return True
        if a1 <= b0 or b1 <= a0:
            return False
    return True


def check_apart(name: str, out: torch.Tensor, other_name: str, other: torch.Tensor, *, same_allowed: bool = False) -> None:
    if same_allowed and out.data_ptr() == other.data_ptr() and out.shape == other.shape and out.stride() == other.stride():
        return
    if overlap(out, other):
        raise ConfigError(f"{name} overlaps {other_name}")


def empty(like: torch.Tensor) -> torch.Tensor:
    """A new contiguous tensor of the same shape, type and device."""
    return torch.empty_like(like, memory_format=torch.contiguous_format)


def rows(t: torch.Tensor) -> tuple[int, int, int]:
    """The fields of a ``_lib.Heads``."""
    token, head, _ = t.stride()
    return t.data_ptr(), token, head


@contextlib.contextmanager
def _elsewhere(index: int):
    with torch.cuda.device(index):  # setting a device up leaves it current
        _lib.ensure_device(index)
        yield


def on_device(index: int):
    """A context in which CUDA device ``index`` is current, and set up. Afterwards the one that was is current again."""
    if torch._C._cuda_getDevice() != index:
        return _elsewhere(index)
    _lib.ensure_device(index)
    return _here


def on_stream(index: int, stream):
    """A context in which ``stream`` (None: the current one) is current, for what a call allocates."""
    if stream is None:
        return _here
    raw(index, stream)
    return torch.cuda.stream(stream)


def raw(index: int, stream) -> int:
    """The handle of ``stream``, or of the device's current one (its number alone: a Stream object costs microseconds)."""
    if stream is None:
        return torch._C._cuda_getCurrentRawStream(index)
    if stream.device.index != index:
        raise ConfigError(f"the stream is on {stream.device}, the tensors on cuda:{index}")
    return stream.cuda_stream
