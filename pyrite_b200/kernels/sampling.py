"""Sampling the next token of each row of logits from given random numbers.

The reference samples one row on the host (temperature and top-p,
pyrite/sampler.py:17-45); greedy is its first index of the largest logit
(sampler.py:12-15).  :func:`sample_rows` does temperature, top-k, top-p and
min-p for every row of a batch on the GPU, each row with its own settings, in
one launch.
"""
from __future__ import annotations

import torch

from .. import _lib
from ._launch import cuda_device, launch, need, need_rows
from .cuda import _check


def sample_rows(logits: torch.Tensor, uniforms: torch.Tensor, temperature: torch.Tensor,
                top_k: torch.Tensor | None = None, top_p: torch.Tensor | None = None,
                min_p: torch.Tensor | None = None, out: torch.Tensor | None = None,
                probs: torch.Tensor | None = None,
                stream: torch.cuda.Stream | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """One token per row of ``logits`` ((rows, vocabulary) float32, at most 2^20 wide).

    ``uniforms``: (rows,) float32 random numbers in [0, 1).  ``temperature``
    (float32; <= 0: greedy), ``top_k`` (int32; <= 0: off), ``top_p`` (float32;
    >= 1: off) and ``min_p`` (float32; <= 0: off): (rows,) each.  In the order
    of falling logits (ties: the lower id first) the kept tokens are those that
    all three filters keep, and the token is the first whose cumulative
    probability exceeds the row's random number.  Returns the ids (int32; -1
    for a row of nothing but -inf and NaN) and their probabilities among the
    kept tokens (float32).
    """
    dev = cuda_device(logits, "logits")
    ld = need_rows(logits, "logits", None, None, dev)
    rows, n = logits.shape
    if rows == 0 or n == 0:
        raise ValueError("logits must have at least one row and one column")
    f32 = torch.float32
    need(uniforms, "uniforms", f32, (rows,), dev)
    need(temperature, "temperature", f32, (rows,), dev)
    for t, name, dt in ((top_k, "top_k", torch.int32), (top_p, "top_p", f32), (min_p, "min_p", f32)):
        if t is not None:
            need(t, name, dt, (rows,), dev)

    def call(st: int) -> tuple[torch.Tensor, torch.Tensor]:
        ids = torch.empty(rows, dtype=torch.int32, device=dev) if out is None else out
        share = torch.empty(rows, dtype=f32, device=dev) if probs is None else probs
        need(ids, "out", torch.int32, (rows,), dev)
        need(share, "probs", f32, (rows,), dev)
        _check(_lib.require().pyrite_cuda_sample_rows(
            logits.data_ptr(), ld, n, rows, uniforms.data_ptr(), temperature.data_ptr(),
            None if top_k is None else top_k.data_ptr(), None if top_p is None else top_p.data_ptr(),
            None if min_p is None else min_p.data_ptr(), ids.data_ptr(), share.data_ptr(), st), "sample rows")
        return ids, share

    return launch(dev, stream, call)
