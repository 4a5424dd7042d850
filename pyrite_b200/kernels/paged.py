"""Serving requests of different lengths over a paged key/value cache.

The reference keeps one contiguous fp32 cache per sequence
(pyrite/executor.py:78-140) and runs one request at a time.  Here the cache of
all requests is a :class:`KVPool` of pages; per decode step

* :func:`page_tables` gives every request the pages its new tokens need and
  the slot of each new token (all on the GPU, from the requests' lengths);
* :func:`append_kv` norms and rotates the new q and k and stores k and v in
  their slots;
* :func:`attention` attends to a prefix that all requests share, read once for
  all of them, and to each request's own tokens.

:func:`store_kv` copies rows of a one-sequence cache (a prefilled prompt) into
slots.  All calls enqueue on the current stream (or ``stream``) and do not
synchronise.  Ids read on the device that lie outside the pool are left out and
reported by :func:`pyrite_b200.kernels.cuda.status` (bit 2).
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from .. import _lib
from ._launch import cuda_device, launch, need, need_list, need_rows
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

    ``lens``, ``new_tokens``: (requests,) int32, tokens held and to come.
    ``free_pages``: (n,) int32 page ids, of which the first ``used`` ((1,)
    int32) are taken; fresh pages follow in request order and ``used_out``
    (default ``used``) receives the new count.  ``table``: (requests, width)
    int32, extended in place.  A request that does not fit (its table row, the
    free pages, ``row_stride`` or the packed capacity) gets no page, slots -1
    and keeps its length; status bit 2 reports it.  ``out`` shares no memory
    with the inputs, and calls that can overlap need one each.
    """
    dev = cuda_device(lens, "lens")
    i32 = torch.int32
    n, capacity = need_list(lens, "lens", i32, dev), need_list(out.slots, "out.slots", i32, dev)
    n_free = need_list(free_pages, "free_pages", i32, dev)
    need(new_tokens, "new_tokens", i32, (n,), dev)
    need(used, "used", i32, (1,), dev)
    need(out.positions, "out.positions", i32, (capacity,), dev)
    need(out.kv_lens, "out.kv_lens", i32, (n,), dev)
    need(out.starts, "out.starts", i32, (n + 1,), dev)
    need(out.ticket, "out.ticket", i32, (1,), dev)
    if table.dtype is not i32 or table.get_device() != dev.index or table.dim() != 2 or table.shape[0] != n or (
            table.stride(1) != 1 and table.shape[1] != 1):
        raise ValueError("table must be an int32 matrix of one row per request, rows contiguous, on the lens' device")
    if used_out is None:
        used_out = used
    else:
        need(used_out, "used_out", i32, (1,), dev)
    if out.kv_lens.data_ptr() in (lens.data_ptr(), new_tokens.data_ptr()):
        raise ValueError("out.kv_lens must not be lens or new_tokens itself")
    width = table.shape[1]
    code = launch(dev, stream, lambda st: _lib.require().pyrite_cuda_page_tables(
        lens.data_ptr(), new_tokens.data_ptr(), n, page_size, free_pages.data_ptr(), n_free, used.data_ptr(),
        used_out.data_ptr(), table.data_ptr(), table.stride(0) if n > 1 else width, width, out.row_stride,
        out.slots.data_ptr(), out.positions.data_ptr(), capacity, out.starts.data_ptr(), out.kv_lens.data_ptr(),
        out.ticket.data_ptr(), st))
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
    dev = cuda_device(qkv, "qkv")
    rows, q_dim = qkv.shape[0], n_heads * HEAD_DIM
    ld = need_rows(qkv, "qkv", None, q_dim + 2 * pool.n_kv_heads * HEAD_DIM, dev)
    if rows == 0 or not 0 <= first <= 0x7FFFFFFF:
        raise ValueError("qkv must have at least one row, and first lie in 0 .. 2^31 - 1")
    if pool.k.get_device() != dev.index:
        raise ValueError("the pool lies on another device")
    need(slots, "slots", torch.int32, (rows,), dev)
    need(positions, "positions", torch.int32, (rows,), dev)
    need(rope, "rope", torch.float64, (rope.shape[0], HEAD_DIM // 2, 2), dev)
    if q_norm is not None:
        need(q_norm, "q_norm", torch.float32, (HEAD_DIM,), dev)
    if k_norm is not None:
        need(k_norm, "k_norm", torch.float32, (HEAD_DIM,), dev)

    def call(st: int) -> torch.Tensor:
        q = torch.empty(rows, q_dim, dtype=torch.float32, device=dev) if q_out is None else q_out
        ldq = need_rows(q, "q_out", rows, q_dim, dev)
        _check(_lib.require().pyrite_cuda_qk_rope_kv_paged(
            qkv.data_ptr(), ld, None if q_norm is None else q_norm.data_ptr(),
            None if k_norm is None else k_norm.data_ptr(), n_heads, pool.n_kv_heads, HEAD_DIM, eps, first,
            positions.data_ptr(), slots.data_ptr(), rows, rope.data_ptr(), rope.shape[0], q.data_ptr(), ldq,
            pool.k.data_ptr(), pool.v.data_ptr(), pool.type_id, pool.n_pages, pool.page_size, st), "append kv")
        return q

    return launch(dev, stream, call)


def store_kv(k: torch.Tensor, v: torch.Tensor, pool: KVPool, slots: torch.Tensor,
             stream: torch.cuda.Stream | None = None) -> None:
    """Rows of one-sequence caches, (rows, n_kv_heads * 128) float32 each with one
    row stride, to the pool's slots (-1: skipped; otherwise each row its own)."""
    dev = cuda_device(k, "k")
    rows = k.shape[0]
    ld = need_rows(k, "k", None, pool.n_kv_heads * HEAD_DIM, dev)
    if need_rows(v, "v", rows, pool.n_kv_heads * HEAD_DIM, dev) != ld:
        raise ValueError("k and v must have one row stride")
    if pool.k.get_device() != dev.index:
        raise ValueError("the pool lies on another device")
    need(slots, "slots", torch.int32, (rows,), dev)
    if rows == 0:
        return
    code = launch(dev, stream, lambda st: _lib.require().pyrite_cuda_kv_store_paged(
        k.data_ptr(), v.data_ptr(), ld, slots.data_ptr(), rows, pool.n_kv_heads, HEAD_DIM, pool.k.data_ptr(),
        pool.v.data_ptr(), pool.type_id, pool.n_pages, pool.page_size, st))
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

    ``q``: (rows, n_heads * 128) float32.  ``prefix_pages``: (pages,) int32,
    of which the first ``prefix_len`` tokens are attended by every row.
    ``table``: (rows, width) int32, each row's own pages (or (width,): one list
    for all rows); ``kv_lens``: (rows,) int32, its own tokens.  A row without
    a token gives zeros.
    """
    dev = cuda_device(q, "q")
    rows = q.shape[0]
    ldq = need_rows(q, "q", None, None, dev)
    if rows == 0 or q.shape[1] == 0 or q.shape[1] % (HEAD_DIM * pool.n_kv_heads):
        raise ValueError("q must be rows of n_heads * 128 values, n_heads a multiple of the pool's KV heads")
    n_heads = q.shape[1] // HEAD_DIM
    if pool.k.get_device() != dev.index:
        raise ValueError("the pool lies on another device")
    need(kv_lens, "kv_lens", torch.int32, (rows,), dev)
    dims = table.dim()
    if table.dtype is not torch.int32 or table.get_device() != dev.index or dims not in (1, 2) or (
            table.stride(-1) != 1 and table.shape[-1] != 1) or (dims == 2 and table.shape[0] != rows):
        raise ValueError("table must be int32, one row per row of q (or one list for all), rows contiguous")
    width = table.shape[-1]
    stride = 0 if dims == 1 else table.stride(0) if rows > 1 else width
    if prefix_len < 0 or (prefix_len > 0 and prefix_pages is None):
        raise ValueError("a prefix needs its pages and a length of at least 0")
    if prefix_len > 0 and need_list(prefix_pages, "prefix_pages", torch.int32, dev) * pool.page_size < prefix_len:
        raise ValueError("prefix_pages hold fewer than prefix_len tokens")

    def call(st: int) -> torch.Tensor:
        o = torch.empty(rows, q.shape[1], dtype=torch.float32, device=dev) if out is None else out
        ldo = need_rows(o, "out", rows, q.shape[1], dev)
        ws = workspace
        if ws is None:
            ws = attention_workspace(rows, n_heads, pool.n_kv_heads, prefix_len, pool.k.dtype, dev)
        elif ws.dtype is not torch.uint8 or ws.get_device() != dev.index or not ws.is_contiguous():
            raise ValueError("workspace must be a contiguous uint8 tensor on q's device")
        _check(_lib.require().pyrite_cuda_attention_paged(
            q.data_ptr(), ldq, pool.k.data_ptr(), pool.v.data_ptr(), pool.type_id, pool.n_pages, pool.page_size,
            prefix_pages.data_ptr() if prefix_len > 0 else None, prefix_len, table.data_ptr(), stride, width,
            kv_lens.data_ptr(), rows, n_heads, pool.n_kv_heads, HEAD_DIM, o.data_ptr(), ldo, ws.data_ptr(),
            ws.numel(), st), "paged attention")
        return o

    return launch(dev, stream, call)
