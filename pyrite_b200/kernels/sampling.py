"""Sampling the next token of each row of logits from given random numbers.

The reference samples one row on the host (temperature and top-p,
pyrite/sampler.py:17-45); greedy is its first index of the largest logit
(sampler.py:12-15).  :func:`sample_rows` does temperature, top-k, top-p and
min-p for every row of a batch on the GPU, each row with its own settings, in
one launch.
"""
from __future__ import annotations

import torch

from ._launch import calls, on
from .cuda import _check


def sample_rows(logits: torch.Tensor, uniforms: torch.Tensor, temperature: torch.Tensor,
                top_k: torch.Tensor | None = None, top_p: torch.Tensor | None = None,
                min_p: torch.Tensor | None = None, out: torch.Tensor | None = None,
                probs: torch.Tensor | None = None,
                stream: torch.cuda.Stream | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """One token per row of ``logits`` ((rows, vocabulary) float32, at most 65535 rows of at most 2^20).

    ``uniforms``: (rows,) float32 random numbers in [0, 1).  ``temperature``
    (float32; <= 0: greedy), ``top_k`` (int32; <= 0: off), ``top_p`` (float32;
    >= 1: off) and ``min_p`` (float32; <= 0: off): (rows,) each.  In the order
    of falling logits (ties: the lower id first) the kept tokens are those that
    all three filters keep, and the token is the first whose cumulative
    probability exceeds the row's random number.  Returns the ids (int32; -1
    for a row of nothing but -inf and NaN) and their probabilities among the
    kept tokens (float32).  A logit further below the row's largest than
    float32's largest number counts as -inf.
    """
    if stream is not None:
        with on(stream, logits):
            return sample_rows(logits, uniforms, temperature, top_k, top_p, min_p, out, probs)
    r = calls().sample_rows(logits, uniforms, temperature, top_k, top_p, min_p, out, probs)
    if type(r) is int:
        _check(r, "sample rows")
    return r
