"""Per-device library contexts and argument plumbing for torch tensors.

PyTorch is used here only for device memory and streams: tensors are passed
to the C ABI as raw device pointers together with torch's current stream.
"""
from __future__ import annotations

import ctypes
import threading

import torch

from . import _lib

_contexts: dict[int, ctypes.c_void_p] = {}
_lock = threading.Lock()


def context(device: int | torch.device | None = None) -> ctypes.c_void_p:
    """Returns (creating once) the library context of a CUDA device."""
    if device is None:
        device = torch.cuda.current_device()
    if isinstance(device, torch.device):
        device = device.index if device.index is not None else torch.cuda.current_device()
    with _lock:
        ctx = _contexts.get(device)
        if ctx is None:
            ctx = ctypes.c_void_p()
            _lib.call("ncm_ctx_create", int(device), ctypes.byref(ctx))
            _contexts[device] = ctx
        return ctx


def release_all() -> None:
    """Destroys every context (the library frees its workspaces)."""
    with _lock:
        for ctx in _contexts.values():
            _lib.load().ncm_ctx_destroy(ctx)
        _contexts.clear()


def stream_of(t: torch.Tensor) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def context_of(device: torch.device) -> ctypes.c_void_p:
    """context() of a tensor's device, without the lock once it exists."""
    return _contexts.get(device.index) or context(device)


def empty_rows(rows: int, width: int, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    """torch.empty((rows, width)), in half its time."""
    return torch.empty_strided((rows, width), (width, 1), dtype=dtype, device=device)


def raw_stream(device: torch.device) -> int:
    """Handle of torch's current stream on a device (the C ABI's stream argument),
    without the stream object that stream_of makes: 0.1 instead of 2.7 us, which
    counts where a call's kernel takes a few microseconds."""
    return torch._C._cuda_getCurrentRawStream(device.index)


def ptr(t: torch.Tensor | None) -> ctypes.c_void_p | None:
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def need(t: torch.Tensor, dtype: torch.dtype, name: str, shape: tuple | None = None) -> torch.Tensor:
    """Validates a device tensor argument (dtype, contiguity, shape)."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    return t


def _refuse_tensor(t, dtype: torch.dtype, name: str, device: torch.device) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}, got {t.device}")


def need_rows(t: torch.Tensor, dtype: torch.dtype, name: str, device: torch.device, width: int) -> int:
    """Validates a [rows, >= width] matrix whose rows may be strided (a column
    slice of a wider matrix, say) and returns its row stride in elements."""
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.device != device:
        _refuse_tensor(t, dtype, name, device)
    shape = t.shape
    if len(shape) != 2 or shape[1] < width:
        raise ValueError(f"{name} must be a matrix of at least {width} columns, got {tuple(shape)}")
    stride, inner = t.stride()
    rows, cols = shape
    if rows <= 1:  # a single row's stride says nothing: the row itself covers what is read
        stride = max(stride, cols + 7 & ~7)
    if (inner != 1 and cols > 1) or stride < cols:
        raise ValueError(f"{name} must have contiguous, separate rows")
    return stride


def need_vec(t: torch.Tensor | None, dtype: torch.dtype, name: str, device: torch.device, n: int | None = None):
    """Address of a contiguous vector argument (None for None), validated."""
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.device != device:
        _refuse_tensor(t, dtype, name, device)
    shape = t.shape
    if len(shape) != 1 or (n is not None and shape[0] != n) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous vector{'' if n is None else f' of {n}'}, got {tuple(shape)}")
    return t.data_ptr()


def sync(device: int | torch.device | None = None) -> None:
    """Waits for torch's current stream and reports device-side failures."""
    dev = torch.device("cuda", device) if isinstance(device, int) else (device or torch.device("cuda"))
    _lib.call("ncm_sync", context(dev), ctypes.c_void_p(torch.cuda.current_stream(dev).cuda_stream))
