"""The native calls of the serving entry points, and their streams.

The checks of the tensors, the choice of the current stream and the launch are
in csrc/serving_calls.cpp: these run on every call of kernels that take a few
microseconds.
"""
from __future__ import annotations

import ctypes
import importlib.machinery
import importlib.util
import threading
from contextlib import contextmanager

import torch

from .. import _lib

_lock = threading.Lock()
_calls = None


def _load():
    from ..build import build_calls, calls_path
    lib, path = _lib.require(), calls_path()
    if not path.is_file():
        try:
            build_calls()
        except Exception as e:
            raise RuntimeError(f"{path.name} is not built; run python -m pyrite_b200.build") from e
    loader = importlib.machinery.ExtensionFileLoader("serving_calls", str(path))
    module = importlib.util.module_from_spec(importlib.util.spec_from_loader("serving_calls", loader))
    loader.exec_module(module)
    for name in module.entries():
        module.bind(name, ctypes.cast(getattr(lib, name), ctypes.c_void_p).value)
    return module


def calls():
    """The module of csrc/serving_calls.cpp, its functions bound to the library."""
    global _calls
    if _calls is None:
        with _lock:
            if _calls is None:
                _calls = _load()
    return _calls


@contextmanager
def on(stream: torch.cuda.Stream, t: torch.Tensor):
    """``stream`` as the current one, so that what a call allocates belongs to the stream it launches on."""
    if stream.device != t.device:
        raise ValueError("the stream belongs to another device than the tensors")
    with torch.cuda.stream(stream):
        yield
