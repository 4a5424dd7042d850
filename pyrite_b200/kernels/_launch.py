"""Argument checks and stream selection of the serving entry points.

These run on every call of kernels that take a few microseconds, so each check
is one expression of tensor attributes on the path where nothing is wrong.
"""
from __future__ import annotations

from contextlib import contextmanager

import torch

try:  # the current stream's handle without building a Stream object (a microsecond and a half)
    from torch._C import _cuda_getCurrentRawStream as _raw_stream
except ImportError:
    def _raw_stream(index: int) -> int:
        return torch.cuda.current_stream(index).cuda_stream


@contextmanager
def _both(device: torch.device, stream: torch.cuda.Stream | None):
    with torch.cuda.device(device):
        if stream is None:
            yield
        else:
            with torch.cuda.stream(stream):
                yield


def launch(device: torch.device, stream: torch.cuda.Stream | None, call) -> None:
    """``call(raw stream)`` with the tensors' device as the current one; what the
    call allocates belongs to the stream that it launches on."""
    if stream is None:
        if torch.cuda.current_device() == device.index:
            return call(_raw_stream(device.index))
    elif stream.device != device:
        raise ValueError("the stream belongs to another device than the tensors")
    with _both(device, stream):
        return call(_raw_stream(device.index))


def need(t: torch.Tensor, what: str, dtype: torch.dtype, shape: tuple[int, ...], device: torch.device) -> None:
    """``t`` is a contiguous tensor of this dtype and shape on ``device`` (a CUDA device with an index)."""
    if t.dtype is not dtype or t.shape != shape or t.get_device() != device.index or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous {dtype} tensor of shape {tuple(shape)} on {device}, got "
                         f"{t.dtype} {tuple(t.shape)} on {t.device}")


def need_list(t: torch.Tensor, what: str, dtype: torch.dtype, device: torch.device) -> int:
    """``t`` is a contiguous vector of this dtype on ``device``; returns its length."""
    if t.dtype is not dtype or t.dim() != 1 or t.get_device() != device.index or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous {dtype} vector on {device}, got {t.dtype} {tuple(t.shape)} on "
                         f"{t.device}")
    return t.shape[0]


def need_rows(t: torch.Tensor, what: str, rows: int | None, cols: int | None, device: torch.device) -> int:
    """``t`` is a float32 matrix with unit stride along its rows; returns its row stride."""
    if t.dtype is torch.float32 and t.get_device() == device.index and t.dim() == 2:
        shape, stride = t.shape, t.stride()
        if (rows is None or shape[0] == rows) and (cols is None or shape[1] == cols) and (stride[1] == 1 or shape[1] == 1):
            return stride[0] if shape[0] > 1 else shape[1]
    raise ValueError(f"{what} must be a float32 matrix of {rows} x {cols} with contiguous rows on {device}, got "
                     f"{t.dtype} {tuple(t.shape)} on {t.device}")


def cuda_device(t: torch.Tensor, what: str) -> torch.device:
    if not t.is_cuda:
        raise ValueError(f"{what} must be a CUDA tensor")
    return t.device
