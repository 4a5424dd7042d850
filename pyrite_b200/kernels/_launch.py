"""Argument checks and stream selection of the serving entry points."""
from __future__ import annotations

from contextlib import contextmanager, nullcontext

import torch


@contextmanager
def _both(device: torch.device, stream: torch.cuda.Stream | None):
    with torch.cuda.device(device):
        if stream is None:
            yield
        else:
            with torch.cuda.stream(stream):
                yield


def launching(device: torch.device, stream: torch.cuda.Stream | None):
    """The context of one call: the tensors' device is the current one, and what
    the call allocates belongs to the stream that it launches on."""
    if stream is not None and stream.device != device:
        raise ValueError("the stream belongs to another device than the tensors")
    if stream is None and torch.cuda.current_device() == device.index:
        return nullcontext()
    return _both(device, stream)


def raw_stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def need(t: torch.Tensor, what: str, dtype: torch.dtype, shape: tuple[int | None, ...], device: torch.device) -> None:
    """``t`` is a contiguous tensor of this dtype and shape (None: any size) on ``device``."""
    if t.dtype != dtype or t.device != device or t.dim() != len(shape) or not t.is_contiguous() or any(
            n is not None and n != m for n, m in zip(shape, t.shape)):
        want = "x".join("?" if n is None else str(n) for n in shape)
        raise ValueError(f"{what} must be a contiguous {dtype} tensor of shape {want} on {device}, got "
                         f"{t.dtype} {tuple(t.shape)} on {t.device}")


def need_rows(t: torch.Tensor, what: str, rows: int | None, cols: int | None, device: torch.device) -> int:
    """``t`` is a float32 matrix with unit stride along its rows; returns its row stride."""
    if t.dtype != torch.float32 or t.device != device or t.dim() != 2 or t.stride(1) != 1 or (
            rows is not None and t.shape[0] != rows) or (cols is not None and t.shape[1] != cols):
        raise ValueError(f"{what} must be a float32 matrix of {rows} x {cols} with contiguous rows on {device}, got "
                         f"{t.dtype} {tuple(t.shape)} on {t.device}")
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def cuda_device(t: torch.Tensor, what: str) -> torch.device:
    if not t.is_cuda:
        raise ValueError(f"{what} must be a CUDA tensor")
    return t.device
