"""Tensor / stream plumbing shared by the kernel wrappers."""
from __future__ import annotations

import contextlib
import ctypes
import importlib.machinery
import importlib.util
import warnings

import torch

from .. import _lib, build

_FAST_SYMBOLS = ("sn_paged_decode_attention", "sn_paged_decode_workspace_size", "sn_rotary_paged_append", "sn_rotary_paged_append_at", "sn_copy_pages",
                 "sn_mamba2_prompt", "sn_mamba2_prompt_workspace_size", "sn_paged_decode_attention_mass",
                 "sn_paged_mass_workspace_size", "sn_evict_positions", "sn_evict_workspace_size", "sn_update_page_bounds", "sn_select_blocks",
                 "sn_select_blocks_workspace_size",
                 "sn_paged_sparse_attention")


class _NoFast:
    """In the place of the short way's functions where it was not built, or
    does not load: every call is left to the wrapper."""
    attend = append = copy = prompt = mass = evict = bounds = select = sparse = staticmethod(lambda *args: None)


_fast = None


def fast():
    """bind/fastcall.cpp, on the loaded library: its functions return None for
    what they leave to the wrappers, an int for a status of the C ABI."""
    global _fast
    if _fast is None:
        lib = _lib.lib()
        path = build.bind_path()
        if not path.exists():
            _fast = _NoFast
            return _fast
        loader = importlib.machinery.ExtensionFileLoader("_fastcall", str(path))
        try:
            m = importlib.util.module_from_spec(importlib.util.spec_from_loader("_fastcall", loader))
            loader.exec_module(m)
        except ImportError as e:
            warnings.warn(f"{path.name} does not load, calls take more host time: {e}")
            _fast = _NoFast
            return _fast
        m.bind({name: ctypes.cast(getattr(lib, name), ctypes.c_void_p).value for name in _FAST_SYMBOLS})
        _fast = m
    return _fast


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
