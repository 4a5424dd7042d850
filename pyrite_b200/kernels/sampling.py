"""Sampling the next token of each row of logits from given random numbers.

The reference samples one row on the host (temperature and top-p,
pyrite/sampler.py:17-45); greedy is its first index of the largest logit
(sampler.py:12-15).  :func:`sample_rows` does temperature, top-k, top-p and
min-p for every row of a batch on the GPU, each row with its own settings, in
one launch.  :func:`token_probs` gives the distributions that it draws from, and
:func:`verify_drafts` compares drafted tokens with them (speculative decoding).
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


def token_probs(logits: torch.Tensor, temperature: torch.Tensor, top_k: torch.Tensor | None = None,
                top_p: torch.Tensor | None = None, min_p: torch.Tensor | None = None, out: torch.Tensor | None = None,
                stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    """The distribution that :func:`sample_rows` draws from with these settings, of each row of ``logits``.

    Returns (rows, vocabulary) float32 (``out``, no view that shares values with
    the logits): each kept token's share, 0 elsewhere; for a greedy row 1 at the
    first index of the largest logit; zeros for a row of nothing but -inf and NaN.
    """
    if stream is not None:
        with on(stream, logits):
            return token_probs(logits, temperature, top_k, top_p, min_p, out)
    r = calls().token_probs(logits, temperature, top_k, top_p, min_p, out)
    if type(r) is int:
        _check(r, "token probs")
    return r


def verify_drafts(probs: torch.Tensor, draft_tokens: torch.Tensor, starts: torch.Tensor, accept: torch.Tensor,
                  pick: torch.Tensor, draft_probs: torch.Tensor | None = None, out: torch.Tensor | None = None,
                  counts: torch.Tensor | None = None,
                  stream: torch.cuda.Stream | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """How many drafted tokens of each request the target accepts, and the token that follows them.

    ``probs``: (rows, vocabulary) float32; the rows of request i are
    ``starts[i]`` to ``starts[i + 1] - 1`` ((requests + 1,) int32, not falling;
    where they do, the entries of shared rows are any of their requests' and
    status bit 2 is set), row t the target's distribution behind t of its drafts
    (:func:`token_probs`), the last one behind all.  ``draft_tokens``: (rows,) int32, entry ``starts[i] + t``
    the draft that follows row t (the last row's is not read; an id outside the
    vocabulary: no draft from here on); ``draft_probs``: (rows, vocabulary) float32, the
    distributions that the drafts were drawn from (None: none, as for tokens
    found by a lookup).  ``accept`` ((rows,) float32) and ``pick`` ((requests,)
    float32): random numbers in [0, 1).  A draft x is accepted while
    ``accept * q(x) < p(x)``; the next token comes from max(p - q, 0) at the
    first refusal, from p behind the last draft, and is the first id whose
    cumulative weight exceeds ``pick`` times the sum.  So the tokens have the
    target's distribution, whatever the drafts are.

    Returns the tokens, (rows,) int32 (``out``, may be ``draft_tokens``, but not a shifted view of them):
    accepted drafts and the next token from ``starts[i]`` on, -1 behind them;
    and their number per request (``counts``).  A request whose row has no
    probability above 0 has no next token.  Entries of no request are left as
    they were (-1 without ``out``).
    """
    if stream is not None:
        with on(stream, probs):
            return verify_drafts(probs, draft_tokens, starts, accept, pick, draft_probs, out, counts)
    r = calls().verify_drafts(probs, draft_tokens, starts, accept, pick, draft_probs, out, counts)
    if type(r) is int:
        _check(r, "verify drafts")
    return r
