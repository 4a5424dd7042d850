"""Serving requests of different lengths over a paged key/value cache.

The reference keeps one contiguous fp32 cache per sequence
(pyrite/executor.py:78-140) and runs one request at a time.  Here the cache of
all requests is a :class:`KVPool` of pages; per decode step

* :func:`page_tables` gives every request the pages its new tokens need and
  the slot of each new token (all on the GPU, from the requests' lengths);
* :func:`append_kv` norms and rotates the new q and k and stores k and v in
  their slots;
* :func:`attention` attends to a prefix that all requests share, read once for
  all of them, and to each request's own tokens;
* :func:`attention_chunks` does that for several new tokens of every request: a
  part of a prompt, or drafted tokens.

:func:`store_kv` copies rows of a one-sequence cache (a prefilled prompt) into
slots.  :func:`fork_requests` makes requests that continue others' (samples of one
prompt, beams), :func:`copy_pages` the copies of pages that they need, and
:func:`release_pages` gives pages of ended requests and refused drafts back.  All calls
enqueue on the current stream (or ``stream``) and do not synchronise.  Ids read on the device that lie outside the pool are left out and
reported by :func:`pyrite_b200.kernels.cuda.status` (bit 2).
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from .. import _lib
from ._launch import calls, on
from .cuda import _check

HEAD_DIM = 128
_TYPE_IDS = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}  # GGML ids


@dataclass
class KVPool:
    """Keys and values in pages: ``(n_pages, n_kv_heads, page_size, 128)`` each,
    float32, float16 or bfloat16; ``page_size`` a power of two, 16 to 256."""

    k: torch.Tensor
    v: torch.Tensor

    def __post_init__(self) -> None:
        k, v = self.k, self.v
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.device != v.device:
            raise ValueError("k and v must be tensors of one shape (n_pages, n_kv_heads, page_size, 128), type and device")
        if not k.is_cuda or not k.is_contiguous() or not v.is_contiguous():
            raise ValueError("k and v must be contiguous CUDA tensors")
        if k.dtype not in _TYPE_IDS:
            raise ValueError("the pool's type must be float32, float16 or bfloat16")
        ps = k.shape[2]
        if k.shape[3] != HEAD_DIM or not 16 <= ps <= 256 or ps & (ps - 1):
            raise ValueError("the head dimension must be 128 and the page size a power of two from 16 to 256")
        if k.shape[0] < 1 or k.shape[1] < 1 or k.shape[0] * ps > 0x7FFFFFFF:
            raise ValueError("the pool must hold 1 to 2^31 - 1 tokens")
        self.type_id = _TYPE_IDS[k.dtype]
        self.n_pages, self.n_kv_heads, self.page_size = k.shape[0], k.shape[1], ps

    @classmethod
    def zeros(cls, n_pages: int, n_kv_heads: int, page_size: int, dtype: torch.dtype = torch.float16,
              device="cuda") -> "KVPool":
        k = torch.zeros(n_pages, n_kv_heads, page_size, HEAD_DIM, dtype=dtype, device=device)
        return cls(k, torch.zeros_like(k))


@dataclass
class TokenSlots:
    """What :func:`page_tables` writes: the new tokens' ``slots`` and
    ``positions`` (request i's at ``i * row_stride``, or packed at
    ``starts[i]`` when ``row_stride`` is 0; -1 elsewhere) and the requests'
    lengths with the new tokens, ``kv_lens``."""

    slots: torch.Tensor      # (capacity,) int32
    positions: torch.Tensor  # (capacity,) int32
    kv_lens: torch.Tensor    # (requests,) int32
    starts: torch.Tensor     # (requests + 1,) int32, packed only
    ticket: torch.Tensor     # (1,) int32, zero between calls
    row_stride: int

    @classmethod
    def empty(cls, requests: int, capacity: int | None = None, row_stride: int = 0, device="cuda") -> "TokenSlots":
        if capacity is None:
            capacity = requests * row_stride
        z = lambda n: torch.zeros(n, dtype=torch.int32, device=device)  # noqa: E731
        return cls(z(capacity), z(capacity), z(requests), z(requests + 1), z(1), row_stride)


def page_tables(lens: torch.Tensor, new_tokens: torch.Tensor, page_size: int, free_pages: torch.Tensor,
                used: torch.Tensor, table: torch.Tensor, out: TokenSlots, used_out: torch.Tensor | None = None,
                stream: torch.cuda.Stream | None = None) -> TokenSlots:
    """Give each request the pages and slots of its new tokens.

    ``lens``, ``new_tokens``: (requests,) int32, tokens held and to come (at
    most 4080 requests).
    ``free_pages``: (n,) int32 page ids, of which the first ``used`` ((1,)
    int32) are taken; fresh pages follow in request order and ``used_out``
    (default ``used``) receives the new count.  ``table``: (requests, width)
    int32, extended in place.  A request that does not fit (its table row, the
    free pages, ``row_stride`` or the packed capacity) gets no page, slots -1
    and keeps its length; status bit 2 reports it, as it does a page id that no
    pool can have, whose tokens get slot -1.  ``out`` shares no memory
    with the inputs, and calls that can overlap need one each.
    """
    if stream is not None:
        with on(stream, lens):
            return page_tables(lens, new_tokens, page_size, free_pages, used, table, out, used_out)
    code = calls().page_tables(lens, new_tokens, page_size, free_pages, used, table,
                               used if used_out is None else used_out, out.slots, out.positions, out.kv_lens,
                               out.starts, out.ticket, out.row_stride)
    if code:
        _check(code, "page tables")
    return out


def append_kv(qkv: torch.Tensor, pool: KVPool, slots: torch.Tensor, positions: torch.Tensor, rope: torch.Tensor,
              n_heads: int, q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None,
              eps: float = 1e-6, first: int = 0, q_out: torch.Tensor | None = None,
              stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    """QK norm (where weights are given), RoPE, and k and v into their slots.

    ``qkv``: (rows, (n_heads + 2 n_kv_heads) * 128) float32, [q | k | v];
    row j sits at position ``first + positions[j]`` of ``rope`` ((max_ctx, 64,
    2) float64 cosines and sines) and in slot ``slots[j]`` (-1: k and v are not
    stored); a negative position skips the row.  Rows of one call have slots
    of their own.  ``q_out`` may be the q part of ``qkv``.  Returns the rotated q.
    """
    if stream is not None:
        with on(stream, qkv):
            return append_kv(qkv, pool, slots, positions, rope, n_heads, q_norm, k_norm, eps, first, q_out)
    q = calls().append_kv(qkv, pool.k, pool.v, slots, positions, rope, n_heads, q_norm, k_norm, eps, first, q_out)
    if type(q) is int:
        _check(q, "append kv")
    return q


def store_kv(k: torch.Tensor, v: torch.Tensor, pool: KVPool, slots: torch.Tensor,
             stream: torch.cuda.Stream | None = None) -> None:
    """Rows of one-sequence caches, (rows, n_kv_heads * 128) float32 each with one
    row stride, to the pool's slots (-1: skipped; otherwise each row its own)."""
    if stream is not None:
        with on(stream, k):
            return store_kv(k, v, pool, slots)
    code = calls().store_kv(k, v, pool.k, pool.v, slots)
    if code:
        _check(code, "store kv")


def attention_workspace(rows: int, n_heads: int, n_kv_heads: int, prefix_len: int = 0,
                        dtype: torch.dtype = torch.float16, device="cuda") -> torch.Tensor:
    """The scratch memory of :func:`attention` for these sizes; calls that can overlap need one each."""
    size = int(_lib.require().pyrite_cuda_attention_paged_workspace_size(rows, n_heads, n_kv_heads, prefix_len,
                                                                         _TYPE_IDS.get(dtype, -1)))
    if size == 0:
        raise ValueError("no attention of these sizes (1..4096 rows, heads a multiple of the KV heads, 128 values each)")
    return torch.empty(size, dtype=torch.uint8, device=device)


def attention(q: torch.Tensor, pool: KVPool, table: torch.Tensor, kv_lens: torch.Tensor,
              prefix_pages: torch.Tensor | None = None, prefix_len: int = 0, out: torch.Tensor | None = None,
              workspace: torch.Tensor | None = None, stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    """Softmax attention of each row of q over the shared prefix and its own tokens.

    ``q``: (rows, n_heads * 128) float32, at most 4096 rows.  ``prefix_pages``: (pages,) int32,
    of which the first ``prefix_len`` tokens are attended by every row.
    ``table``: (rows, width) int32, each row's own pages (or (width,): one list
    for all rows); ``kv_lens``: (rows,) int32, its own tokens.  A row without
    a token gives zeros.
    """
    if stream is not None:
        with on(stream, q):
            return attention(q, pool, table, kv_lens, prefix_pages, prefix_len, out, workspace)
    o = calls().attention(q, pool.k, pool.v, table, kv_lens, prefix_pages, prefix_len, out, workspace)
    if type(o) is int:
        _check(o, "paged attention")
    return o


def chunks_workspace(rows: int, requests: int, n_heads: int, n_kv_heads: int, dtype: torch.dtype = torch.float16,
                     device="cuda") -> torch.Tensor:
    """The scratch memory of :func:`attention_chunks` for these sizes; calls that can overlap need one each."""
    size = int(_lib.require().pyrite_cuda_attention_chunks_workspace_size(rows, requests, n_heads, n_kv_heads,
                                                                          _TYPE_IDS.get(dtype, -1)))
    if size == 0:
        raise ValueError("no attention of these sizes (1..2^20 rows, 1..4080 requests, heads a multiple of the KV heads, "
                         "at most 1024)")
    return torch.empty(size, dtype=torch.uint8, device=device)


def attention_chunks(q: torch.Tensor, pool: KVPool, table: torch.Tensor, starts: torch.Tensor, kv_lens: torch.Tensor,
                     prefix_pages: torch.Tensor | None = None, prefix_len: int = 0, out: torch.Tensor | None = None,
                     workspace: torch.Tensor | None = None, stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    """Softmax attention of several new tokens of every request, each over the tokens before it and itself.

    ``q``: (rows, n_heads * 128) float32, packed: request i's new tokens are
    the rows ``starts[i]`` to ``starts[i + 1] - 1`` ((requests + 1,) int32, not
    falling; :attr:`TokenSlots.starts`) and the last of its ``kv_lens[i]``
    tokens ((requests,) int32; :attr:`TokenSlots.kv_lens`), whose keys and
    values are in the pool.  Every row attends to the prefix, as in
    :func:`attention`, and to its request's own tokens up to itself, in the
    pages of ``table`` ((requests, width) int32).  A row without a token gives
    zeros; rows of no request are left as they were (zeros without ``out``).
    ``out`` may be ``q`` itself, but no other view that shares values with it.
    Scores have to lie within float32's range, values times the number of
    tokens below 2^113; an infinite or NaN value makes its column infinite or
    NaN in the rows that see it.
    At most 2^20 rows of 4080 requests.
    """
    if stream is not None:
        with on(stream, q):
            return attention_chunks(q, pool, table, starts, kv_lens, prefix_pages, prefix_len, out, workspace)
    o = calls().attention_chunks(q, pool.k, pool.v, table, starts, kv_lens, prefix_pages, prefix_len, out, workspace)
    if type(o) is int:
        _check(o, "attention of chunks")
    return o


def fork_requests(parents: torch.Tensor, lens: torch.Tensor, page_size: int, free_pages: torch.Tensor,
                  used: torch.Tensor, table: torch.Tensor, shared: torch.Tensor, copies: torch.Tensor | None = None,
                  lens_out: torch.Tensor | None = None, used_out: torch.Tensor | None = None,
                  shared_out: torch.Tensor | None = None, stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    """Make requests that continue others'.

    Request i with ``parents[i] >= 0`` ((requests,) int32), which holds
    nothing (``lens[i]`` 0), continues request ``parents[i]``, itself not
    forked in this call: they share its full pages, and a partly filled last
    one gets a copy in a page of its own.  ``free_pages``, ``used`` and
    ``table`` as in :func:`page_tables`; ``shared``: (n_pages,) int32, the
    holders of each page beside the first (zeros to begin with).  ``lens_out``,
    ``used_out`` and ``shared_out`` default to ``lens``, ``used`` and
    ``shared``.  Returns the pages to copy, (2, requests) int32 (``copies``):
    sources and destinations, -1 where there is none, for :func:`copy_pages`.
    A request that cannot be served keeps its length and sets status bit 2.
    """
    if stream is not None:
        with on(stream, lens):
            return fork_requests(parents, lens, page_size, free_pages, used, table, shared, copies, lens_out, used_out,
                                 shared_out)
    c = calls().fork_requests(parents, lens, page_size, free_pages, used, table, shared, copies,
                              lens if lens_out is None else lens_out, used if used_out is None else used_out,
                              shared if shared_out is None else shared_out)
    if type(c) is int:
        _check(c, "fork requests")
    return c


def copy_pages(pools: list[KVPool], copies: torch.Tensor, stream: torch.cuda.Stream | None = None) -> None:
    """Whole pages ``copies[0, i]`` to ``copies[1, i]`` ((2, n) int32; -1: no copy) in every pool.

    ``pools``: pools of one shape and type, one per layer.  No page may be a
    destination twice, or a source and a destination.
    """
    if stream is not None:
        with on(stream, copies):
            return copy_pages(pools, copies)
    code = calls().copy_pages([p.k for p in pools], [p.v for p in pools], copies)
    if code:
        _check(code, "copy pages")


def release_pages(lens: torch.Tensor, keep: torch.Tensor, page_size: int, free_pages: torch.Tensor, used: torch.Tensor,
                  table: torch.Tensor, shared: torch.Tensor, lens_out: torch.Tensor | None = None,
                  used_out: torch.Tensor | None = None, shared_out: torch.Tensor | None = None,
                  stream: torch.cuda.Stream | None = None) -> None:
    """Cut every request back to its first ``keep[i]`` tokens ((requests,) int32; 0: it ends).

    A page that no request holds any more goes back to ``free_pages``, in
    ascending order in front of the free ones, and ``used`` falls; a page that
    others still hold has its count in ``shared`` lowered.  ``lens`` becomes
    min(keep, lens).  Arguments and outputs otherwise as in
    :func:`fork_requests`; the table is not changed.  A request that is to
    grow again inside a page that others hold has to be forked first.
    """
    if stream is not None:
        with on(stream, lens):
            return release_pages(lens, keep, page_size, free_pages, used, table, shared, lens_out, used_out, shared_out)
    code = calls().release_pages(lens, keep, page_size, free_pages, used, table, shared,
                                 lens if lens_out is None else lens_out, used if used_out is None else used_out,
                                 shared if shared_out is None else shared_out)
    if code:
        _check(code, "release pages")
