"""Tensor / stream plumbing shared by the kernel wrappers."""
from __future__ import annotations

import contextlib

import torch

from .. import _lib


def stream_handle(stream=None) -> int:
    """Raw cudaStream_t for `stream` (None -> torch's current stream)."""
    if stream is None:
        return torch.cuda.current_stream().cuda_stream
    if isinstance(stream, torch.cuda.Stream):
        return stream.cuda_stream
    if isinstance(stream, int):
        return stream
    h = getattr(stream, "cuda_stream", None)
    if h is not None:
        return int(h)
    raise TypeError(f"cannot interpret {type(stream).__name__} as a CUDA stream")


@contextlib.contextmanager
def _on_other_stream(stream, h: int):
    with torch.cuda.stream(stream if isinstance(stream, torch.cuda.Stream) else torch.cuda.ExternalStream(h)):
        yield h


def current_handle(device: int) -> int:
    """stream_handle(None) for the current device `device`, without a Stream
    object around it (a short call spends most of its time on the host)."""
    return torch._C._cuda_getCurrentRawStream(device)


def on_stream(stream=None):
    """A context that makes `stream` (as stream_handle takes it) torch's
    current stream, so that what a wrapper allocates belongs to the stream its
    kernels run on, and gives the raw handle."""
    h = stream_handle(stream)
    if h == torch.cuda.current_stream().cuda_stream:
        return contextlib.nullcontext(h)
    return _on_other_stream(stream, h)


def same_device(**tensors) -> None:
    """Every given tensor (or None) is on torch's current CUDA device, where the kernels launch."""
    cur = torch.cuda.current_device()
    for name, t in tensors.items():
        if t is not None and t.device.index != cur:
            raise ValueError(f"{name} is on {t.device}, but the current CUDA device is cuda:{cur}")


def require_cuda(name: str, t: torch.Tensor, dtype=None, dim=None) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (sonata_b200 has no CPU path)")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if dim is not None and t.dim() != dim:
        raise ValueError(f"{name} must be {dim}-D, got shape {tuple(t.shape)}")


def row_major(name: str, t: torch.Tensor) -> int:
    """Row stride of a 2-D tensor whose last dim is contiguous."""
    if t.stride(-1) != 1:
        raise ValueError(f"{name} must have a contiguous last dimension")
    return t.stride(0) if t.size(0) > 1 else max(t.stride(0), t.size(1))


def call(fn: str, *args) -> None:
    _lib.call(fn, *args)
