"""The paged cache on a B200: block tables and slot maps, the append, attention.

Oracles: a host loop for the tables; fp64 numpy / torch for the append and the
attention.  The cache values are given in the cache's own type, so rounding
them is not part of the attention's error.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

HD = 128
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def K(cuda_device):
    from pyrite_b200.kernels import cuda
    cuda.status()
    return cuda


@pytest.fixture(scope="module")
def paged(cuda_device):
    from pyrite_b200.kernels import paged
    return paged


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def pages_of(n, ps):
    return -(-n // ps)


# ---- block tables and slot maps ----------------------------------------------------------
def host_tables(lens, new, ps, free, used, table, capacity, row_stride):
    table, avail = table.copy(), len(free) - used
    slots, pos = np.full(capacity, -1), np.full(capacity, -1)
    kv, starts, first, taken, fits = [], [0], 0, 0, True
    for i, (n, t) in enumerate(zip(lens, new)):
        ok = n >= 0 and t >= 0 and n + t <= table.shape[1] * ps and (row_stride == 0 or t <= row_stride)
        need = pages_of(n + t, ps) - pages_of(n, ps) if ok else 0
        served = ok and (need == 0 or first + need <= avail)
        # packed places end at capacity: a request that passes it is not served
        places = sum(max(x, 0) for x in new[:i + 1])
        served = served and (row_stride > 0 or t == 0 or places <= capacity)
        if served:
            for p in range(need):
                table[i, pages_of(n, ps) + p] = free[used + first + p]
            if need:
                taken = first + need
        first += need
        at = i * row_stride if row_stride else starts[-1]
        for j in range(t if served else 0):
            if at + j < capacity:
                slots[at + j], pos[at + j] = table[i, (n + j) // ps] * ps + (n + j) % ps, n + j
        starts.append(min(capacity, starts[-1] + max(t, 0)))
        kv.append(n + t if served else max(n, 0))
        fits = fits and served
    if row_stride == 0:
        fits = fits and sum(max(t, 0) for t in new) <= capacity
    return table, slots, pos, np.array(kv), np.array(starts), used + taken, fits


def run_tables(paged, K, lens, new, ps, width, n_free, row_stride, capacity, seed=0, alias=False):
    rng = np.random.default_rng(seed)
    n = len(lens)
    free = rng.permutation(n_free + 5)[:n_free].astype(np.int32)
    table, used = np.full((n, width), -1, dtype=np.int32), 0
    for i, m in enumerate(lens):
        p = min(pages_of(max(m, 0), ps), width)
        p = min(p, n_free - used)
        table[i, :p] = free[used:used + p]
        used += p
    want = host_tables(lens, new, ps, free, used, table.astype(np.int64), capacity, row_stride)
    # one guard column and guard words behind every output
    big = torch.full((n, width + 1), -7, dtype=torch.int32, device="cuda")
    big[:, :width] = torch.from_numpy(table)
    out = paged.TokenSlots.empty(n, capacity=capacity, row_stride=row_stride)
    d_used = ints([used])
    d_out = d_used if alias else ints([-9])
    paged.page_tables(ints(lens), ints(new), ps, torch.from_numpy(free).cuda(), d_used, big[:, :width], out,
                      used_out=None if alias else d_out)
    torch.cuda.synchronize()
    status = K.status()
    assert np.array_equal(big[:, :width].cpu().numpy(), want[0])
    assert bool((big[:, width] == -7).all())
    assert np.array_equal(out.slots.cpu().numpy(), want[1])
    assert np.array_equal(out.positions.cpu().numpy(), want[2])
    assert np.array_equal(out.kv_lens.cpu().numpy(), want[3])
    if row_stride == 0:
        assert np.array_equal(out.starts.cpu().numpy(), want[4])
    assert int(d_out) == want[5] and int(out.ticket) == 0
    if not alias:
        assert int(d_used) == used
    assert status == (0 if want[6] else 4)
    return want


@pytest.mark.parametrize("n,ps,held,new,row_stride", [
    (1, 16, 0, 1, 1), (1, 16, 16, 1, 1), (16, 16, 500, 1, 1), (7, 64, 200, 3, 3), (128, 32, 900, 1, 1),
    (1, 16, 0, 1, 0), (5, 16, 33, 40, 0), (128, 16, 900, 700, 0), (33, 128, 1000, 300, 0), (4080, 16, 50, 9, 0),
    (4080, 256, 600, 1, 1), (2, 16, 0, 20000, 0)])
def test_tables_match_the_host_loop(paged, K, n, ps, held, new, row_stride):
    rng = np.random.default_rng(n * 131 + ps)
    lens = rng.integers(0, held + 1, n).tolist()
    fresh = rng.integers(0, new + 1, n).tolist()
    width = pages_of(held + new, ps) + 1
    n_free = sum(pages_of(a + b, ps) for a, b in zip(lens, fresh)) + 3
    cap = n * row_stride if row_stride else max(1, sum(fresh) + 13)
    assert run_tables(paged, K, lens, fresh, ps, width, n_free, row_stride, cap, alias=bool(n % 2))[6]


def test_tables_requests_that_do_not_fit(paged, K):
    # too long for its row; negative sizes; more new tokens than the row stride
    run_tables(paged, K, [10, 60, -3, 5, 20], [3, 9, 2, -1, 2], 16, 4, 40, 0, 30)
    run_tables(paged, K, [10, 60, -3, 5, 20, 0], [3, 4, 2, -1, 5, 4], 16, 4, 40, 4, 24)
    # the free list runs out in the middle: later requests that need a page are left out, others not
    want = run_tables(paged, K, [15, 16, 16, 3, 32], [1, 1, 40, 2, 1], 16, 8, 9, 0, 60, alias=True)
    assert not want[6] and want[3].tolist() == [16, 17, 16, 5, 32]
    # packed places end at capacity
    run_tables(paged, K, [0, 4, 9], [5, 6, 7], 16, 4, 20, 0, 13)
    # nothing left at all, nothing needed
    run_tables(paged, K, [3, 7], [1, 2], 16, 2, 2, 0, 3)
    run_tables(paged, K, [0, 0], [0, 0], 16, 2, 2, 1, 2)
    assert K.status() == 0


def test_tables_packed_places_past_capacity(paged, K):
    """A request whose places end past capacity takes no page and keeps its length, like every later
    one with new tokens; one without new tokens is served."""
    want = run_tables(paged, K, [0, 20, 9, 30, 33], [5, 12, 7, 0, 1], 16, 4, 20, 0, 16)
    assert want[3].tolist() == [5, 20, 9, 30, 33] and want[4].tolist() == [0, 5, 16, 16, 16, 16]
    run_tables(paged, K, [0, 0, 0], [40, 3, 0], 16, 4, 20, 0, 8, alias=True)  # the first alone is too many
    run_tables(paged, K, [5], [9], 16, 4, 20, 0, 8)
    run_tables(paged, K, [5], [9], 16, 4, 20, 0, 9)
    n = 4080  # several blocks: the last requests do not fit
    want = run_tables(paged, K, [3] * n, [20] * n, 16, 3, 2 * n, 0, 20 * n - 50, alias=True)
    assert want[3].tolist() == [23] * (n - 3) + [3] * 3
    assert K.status() == 0


def test_tables_refuse_lengths_written_over_their_inputs(paged, K):
    n = 5
    lens, fresh = ints([0] * n), ints([1] * n)
    out = paged.TokenSlots.empty(n, row_stride=1)
    table = torch.full((n, 2), -1, dtype=torch.int32, device="cuda")
    for t in (lens, fresh):
        out.kv_lens = t
        with pytest.raises(ValueError, match="kv_lens"):
            paged.page_tables(lens, fresh, 16, ints(range(20)), ints([0]), table, out)
    out.kv_lens = ints([0] * n)
    with pytest.raises(ValueError, match="shape"):
        paged.page_tables(lens, fresh, 48, ints(range(20)), ints([0]), table, out)
    torch.cuda.synchronize()
    assert K.status() == 0 and bool((table == -1).all())


@pytest.mark.parametrize("rows", [1, 17, 400])
def test_append_rotates_q_in_place(paged, K, rows):
    """q_out may be the q part of qkv: the same q and the same keys as with rows of its own."""
    nq, nkv, ps = 6, 2, 16
    qkv = torch.randn(rows, (nq + 2 * nkv) * HD, device="cuda")
    pools = [paged.KVPool.zeros(pages_of(rows, ps), nkv, ps, torch.float16) for _ in range(2)]
    slots = torch.randperm(rows, device="cuda").to(torch.int32)
    pos = torch.arange(rows, dtype=torch.int32, device="cuda")
    w = torch.rand(2, HD, device="cuda") + 0.5
    want = paged.append_kv(qkv, pools[0], slots, pos, rope_table(rows), nq, q_norm=w[0], k_norm=w[1])
    rest = qkv[:, nq * HD:].clone()
    got = paged.append_kv(qkv, pools[1], slots, pos, rope_table(rows), nq, q_norm=w[0], k_norm=w[1],
                          q_out=qkv[:, :nq * HD])
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(qkv[:, nq * HD:], rest)
    assert torch.equal(pools[0].k, pools[1].k) and torch.equal(pools[0].v, pools[1].v)
    for first in (-1, 2 ** 31, 2 ** 32):
        with pytest.raises(ValueError, match="first"):
            paged.append_kv(qkv, pools[0], slots, pos, rope_table(rows), nq, first=first)


def test_tables_wants_far_past_the_free_list(paged, K):
    """Requests whose pages add up to many times the list (19 free): those that need one are left out."""
    want = run_tables(paged, K, [0, 5, 0, 16, 0], [20 * 16, 3, 300 * 16, 1, 900 * 16], 16, 1000, 21, 0, 25000)
    assert want[3].tolist() == [0, 8, 0, 16, 0]
    n = 4080
    want = run_tables(paged, K, [0] * n, [256] * n, 16, 20, 40, 256, n * 256, alias=True)
    assert want[3].sum() == 2 * 256 and want[5] == 32
    assert K.status() == 0


def test_tables_replayed_in_a_graph(paged, K):
    """The same captured call step after step: lengths grow on the device, the page count in place."""
    ps, width, n = 16, 6, 9
    lens, fresh = ints([0, 3, 15, 16, 17, 31, 32, 60, 5]), ints([1, 1, 1, 0, 1, 1, 1, 1, 1])
    table = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
    free = torch.randperm(n * width, device="cuda").to(torch.int32)
    used = 0
    for i, m in enumerate(lens.tolist()):
        p = pages_of(m, ps)
        table[i, :p] = free[used:used + p]
        used += p
    used = ints([used])
    host = [lens.tolist(), table.cpu().numpy().astype(np.int64), int(used)]
    out = paged.TokenSlots.empty(n, row_stride=1)
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        paged.page_tables(lens, fresh, ps, free, used, table, out)
        lens.copy_(out.kv_lens)
    for _ in range(25):
        graph.replay()
        host[1], slots, _, kv, _, host[2], ok = host_tables(host[0], fresh.tolist(), ps, free.tolist(), host[2],
                                                            host[1], n, 1)
        host[0] = kv.tolist()
        assert ok and out.slots.tolist() == slots.tolist()
        assert lens.tolist() == host[0] and int(used) == host[2]
    assert np.array_equal(table.cpu().numpy(), host[1]) and K.status() == 0


# ---- append -------------------------------------------------------------------------------
def rope_table(n, theta=1e6):
    inv = theta ** (-2.0 * np.arange(64) / HD)
    ang = np.arange(n)[:, None] * inv[None, :]
    return torch.from_numpy(np.ascontiguousarray(np.stack([np.cos(ang), np.sin(ang)], -1))).cuda()


def near(got, want, t):
    """got is want (fp64) rounded once to t: half a step, plus the fp64 arithmetic's own error."""
    fi = torch.finfo(t)
    tol = want.abs() * (fi.eps / 2) * (1 + 1e-6) + fi.smallest_normal * fi.eps + 1e-14
    assert bool(((got.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,nq,nkv,norm,ps", [(1, 2, 1, False, 16), (5, 12, 3, True, 32), (300, 16, 8, True, 64),
                                                 (17, 64, 4, False, 256), (3, 3, 3, True, 16)])
def test_append(paged, K, dtype, rows, nq, nkv, norm, ps):
    t, max_ctx, first = DTYPES[dtype], 5000, 7
    g = torch.Generator(device="cuda").manual_seed(rows * 7 + nq)
    width = (nq + 2 * nkv) * HD
    qkv = torch.randn(rows, width + 6, generator=g, device="cuda")[:, :width]  # a row stride of its own
    pool = paged.KVPool.zeros(pages_of(rows, ps) + 2, nkv, ps, t)
    pool.k.fill_(3.0)
    pool.v.fill_(5.0)
    slots = torch.randperm(pool.n_pages * ps, generator=g, device="cuda")[:rows].to(torch.int32)
    pos = torch.randint(0, max_ctx - first, (rows,), generator=g, device="cuda", dtype=torch.int32)
    if rows > 2:
        slots[1], pos[2] = -1, -1
        slots[2] = -1
    qn, kn = (torch.rand(2, HD, generator=g, device="cuda") + 0.5) if norm else (None, None)
    rope = rope_table(max_ctx)
    q_out = torch.full((rows, nq * HD + 2), 9.0, device="cuda")
    paged.append_kv(qkv, pool, slots, pos, rope, nq, q_norm=qn, k_norm=kn, eps=1e-5, first=first,
                    q_out=q_out[:, :nq * HD])
    torch.cuda.synchronize()
    assert K.status() == 0
    x = qkv.double().reshape(rows, nq + 2 * nkv, HD)
    q, k, v = x[:, :nq], x[:, nq:nq + nkv], x[:, nq + nkv:]
    if norm:
        q = q / (q.square().mean(-1, keepdim=True) + 1e-5).sqrt() * qn.double()
        k = k / (k.square().mean(-1, keepdim=True) + 1e-5).sqrt() * kn.double()
    cs = rope[(pos.long() + first).clamp(min=0)][:, None]

    def rot(y):
        a, b = y[..., :64], y[..., 64:]
        return torch.cat([a * cs[..., 0] - b * cs[..., 1], a * cs[..., 1] + b * cs[..., 0]], -1)

    on = pos >= 0
    near(q_out[on, :nq * HD], rot(q)[on].reshape(-1, nq * HD), torch.float32)
    assert bool((q_out[~on] == 9.0).all()) and bool((q_out[:, nq * HD:] == 9.0).all())
    wk, wv = torch.full_like(pool.k, 3.0).double(), torch.full_like(pool.v, 5.0).double()
    s = slots.long()[slots >= 0]
    wk[s // ps, :, s % ps], wv[s // ps, :, s % ps] = rot(k)[slots >= 0], v[slots >= 0]
    near(pool.k, wk, t)
    near(pool.v, wv, t)


def test_append_and_store_leave_out_slots_past_the_pool(paged, K):
    pool = paged.KVPool.zeros(2, 1, 16, torch.float16)
    x = torch.randn(3, 3 * HD, device="cuda")
    paged.append_kv(x, pool, ints([32, 5, 2 ** 31 - 1]), ints([0, 1, 2]), rope_table(8), 1)
    torch.cuda.synchronize()
    assert K.status() == 4
    live = pool.v.float().abs().sum(-1).view(-1) > 0
    assert live.nonzero().flatten().tolist() == [5]
    paged.append_kv(x, pool, ints([1, 2, 3]), ints([0, 8, 7]), rope_table(8), 1)  # position 8 of a table of 8
    torch.cuda.synchronize()
    assert K.status() == 4 and not bool(pool.v[0, 0, 2].any()) and bool(pool.v[0, 0, 3].any())
    paged.store_kv(x[:, :HD], x[:, HD:2 * HD], pool, ints([40, 9, -1]))
    torch.cuda.synchronize()
    assert K.status() == 4
    assert torch.equal(pool.k[0, 0, 9], x[1, :HD].half()) and torch.equal(pool.v[0, 0, 9], x[1, HD:2 * HD].half())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_store(paged, K, dtype):
    t = DTYPES[dtype]
    pool = paged.KVPool.zeros(5, 3, 32, t)
    cache = torch.randn(2, 70, 3 * HD, device="cuda")
    slots = torch.randperm(160, device="cuda")[:70].to(torch.int32)
    paged.store_kv(cache[0], cache[1], pool, slots)
    torch.cuda.synchronize()
    s = slots.long()
    assert torch.equal(pool.k[s // 32, :, s % 32], cache[0].view(70, 3, HD).to(t))
    assert torch.equal(pool.v[s // 32, :, s % 32], cache[1].view(70, 3, HD).to(t))
    assert K.status() == 0


# ---- attention ------------------------------------------------------------------------------
class Case:
    """Pools of random pages, tables and lengths; the pages outside every request hold NaN."""

    def __init__(self, paged, rows, nq, nkv, prefix, lens, ps, t, seed=0, scale=1.4, slack=1):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.rows, self.nq, self.nkv, self.prefix, self.ps, self.lens_host = rows, nq, nkv, prefix, ps, list(lens)
        shared = pages_of(prefix, ps)
        total = shared + sum(pages_of(n, ps) for n in lens) + 3
        ids = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
        shape = (total, nkv, ps, HD)
        k = torch.randn(shape, generator=g, device="cuda").mul_(scale)
        v = torch.randn(shape, generator=g, device="cuda")
        width = max([pages_of(n, ps) for n in lens] + [0]) + slack
        table = torch.full((rows, width), -1, dtype=torch.int32, device="cuda")
        used, free, at = torch.zeros(total, ps, dtype=torch.bool, device="cuda"), ids.tolist(), shared
        self.pre_ids = free[:shared]
        for i, p in enumerate(self.pre_ids):
            used[p, :min(ps, prefix - i * ps)] = True
        self.own_ids = []
        for j, n in enumerate(lens):
            own = free[at:at + pages_of(n, ps)]
            at += len(own)
            self.own_ids.append(own)
            if own:
                table[j, :len(own)] = ints(own)
            for i, p in enumerate(own):
                used[p, :min(ps, n - i * ps)] = True
        k.masked_fill_(~used[:, None, :, None], float("nan"))  # what no request holds is never read into a result
        v.masked_fill_(~used[:, None, :, None], float("nan"))
        self.pool = paged.KVPool(k.to(t), v.to(t))
        self.q = torch.randn(rows, nq * HD, generator=g, device="cuda").mul_(scale)
        self.table, self.lens, self.pre = table, ints(list(lens)), ints(self.pre_ids)

    def call(self, paged, **kw):
        return paged.attention(self.q, self.pool, self.table, self.lens,
                               prefix_pages=self.pre if self.prefix else None, prefix_len=self.prefix, **kw)

    def gather(self, pool, b):
        def tok(ids, n):
            if n == 0:
                return torch.zeros(self.nkv, 0, HD, dtype=torch.float64, device="cuda")
            return torch.cat([pool[p] for p in ids], 1)[:, :n].double()
        return torch.cat([tok(self.pre_ids, self.prefix), tok(self.own_ids[b], self.lens_host[b])], 1)

    def oracle(self):
        """fp64 result and, per value, sum_t p_t |v_t|."""
        want = torch.zeros(self.rows, self.nq, HD, dtype=torch.float64, device="cuda")
        mag = torch.zeros_like(want)
        grp = self.nq // self.nkv
        for b in range(self.rows):
            k, v = self.gather(self.pool.k, b), self.gather(self.pool.v, b)
            if k.shape[1] == 0:
                continue
            q = self.q[b].double().view(self.nkv, grp, HD)
            p = torch.softmax(torch.einsum("hgd,htd->hgt", q, k) / math.sqrt(HD), -1)
            want[b] = torch.einsum("hgt,htd->hgd", p, v).reshape(self.nq, HD)
            mag[b] = torch.einsum("hgt,htd->hgd", p, v.abs()).reshape(self.nq, HD)
        return want.view(self.rows, -1), mag.view(self.rows, -1)

    def check(self, got, tol=1e-4, rms=5e-6):
        # Worst value: the bar of the decode attention's own test, 1e-4 of sum p |v|.  Root mean square: a score
        # is a sum of 128 products, ~14 in magnitude sum at this scale, with roundings of 2^-24 each in at most 16
        # steps and, in 16-bit caches, a split of q and p into planes of at least 17 bits: under 4e-6 relative.
        want, mag = self.oracle()
        err = (got.double() - want).abs()
        assert bool((err <= tol * mag + 1e-30).all()), float((err / (mag + 1e-30)).max())
        if want.numel() and float(want.abs().max()) > 0:
            assert float(err.square().mean().sqrt() / want.square().mean().sqrt()) <= rms


SHAPES = [  # rows, q heads, kv heads, prefix, own lengths, page
    (1, 1, 1, 0, [1], 16),
    (1, 16, 8, 0, [97], 16),
    (1, 32, 8, 1, [0], 16),
    (2, 8, 8, 15, [0, 16], 16),
    (3, 12, 3, 16, [1, 0, 17], 16),
    (3, 40, 4, 129, [5, 64, 300], 64),
    (16, 16, 8, 250, [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 100, 127, 128, 129, 200], 16),
    (5, 64, 4, 1000, [700, 3, 0, 250, 64], 128),
    (4, 32, 4, 0, [0, 0, 0, 0], 16),
    (4, 32, 4, 0, [0, 1, 0, 2000], 256),
    (33, 32, 8, 511, [7] * 33, 32),
    (70, 8, 2, 70, list(range(70)), 16),
    (2, 6, 2, 3, [4000, 5], 16),
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[0]}r{s[1]}q{s[2]}k{s[3]}p")
def test_attention(paged, K, shape, dtype):
    rows, nq, nkv, prefix, lens, ps = shape
    c = Case(paged, rows, nq, nkv, prefix, lens, ps, DTYPES[dtype], seed=rows + prefix)
    got = c.call(paged)
    torch.cuda.synchronize()
    assert K.status() == 0
    c.check(got)
    empty = [j for j in range(rows) if prefix == 0 and lens[j] == 0]
    assert bool((got[empty] == 0).all())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,nq,nkv,prefix,ps", [
    (8, 16, 4, 256, 16), (8, 16, 4, 257, 64), (32, 8, 8, 1024, 256), (40, 32, 2, 383, 16), (17, 24, 3, 640, 128),
    (130, 4, 2, 1025, 32), (2, 128, 4, 900, 16), (3, 20, 2, 300, 16),
    (64, 32, 4, 256, 16), (64, 32, 4, 257, 64), (130, 16, 4, 383, 32), (33, 64, 4, 640, 128), (300, 8, 2, 1025, 256),
    (50, 1, 1, 11000, 16)])
def test_attention_prefix_tiles(paged, K, dtype, rows, nq, nkv, prefix, ps):
    """Prefixes of whole and broken tiles, one and several tiles of query rows, with and without own keys."""
    for lens in ([0] * rows, [(7 * j) % 41 for j in range(rows)]):
        c = Case(paged, rows, nq, nkv, prefix, lens, ps, DTYPES[dtype], seed=prefix + rows)
        got = c.call(paged)
        torch.cuda.synchronize()
        assert K.status() == 0
        c.check(got)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,prefix", [(3, 64), (16, 700), (64, 700)])
def test_attention_leaves_out_bad_prefix_pages(paged, K, dtype, rows, prefix):
    c = Case(paged, rows, 16, 4, prefix, [j % 5 for j in range(rows)], 16, DTYPES[dtype], seed=2)
    keep = list(c.pre_ids)
    c.pre[1], c.pre[-1] = -1, 2 ** 31 - 1  # keys 16 .. 31 and the last page's
    got = c.call(paged)
    torch.cuda.synchronize()
    assert K.status() == 4
    last = (prefix - 1) // 16 * 16
    gone = torch.zeros(prefix, dtype=torch.bool)
    gone[16:32] = True
    gone[last:] = True

    def gather(pool, b):
        pre = torch.cat([pool[p] for p in keep], 1)[:, :prefix].double()[:, ~gone]
        own = [pool[p] for p in c.own_ids[b]]
        n = c.lens_host[b]
        return torch.cat([pre] + ([torch.cat(own, 1)[:, :n].double()] if n else []), 1)

    c.gather = gather
    c.check(got)


def test_attention_on_two_streams_at_once(paged, K):
    """Two calls in flight, each with a workspace of its own, many times over."""
    cases = [Case(paged, 16, 32, 4, n, list(range(0, 320, 20)), 16, torch.float16, seed=s) for s, n in ((1, 600), (2, 1500))]
    want = [c.call(paged).clone() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    outs = [[torch.empty_like(w) for _ in range(6)] for w in want]
    ws = [paged.attention_workspace(16, 32, 4, c.prefix, torch.float16) for c in cases]
    torch.cuda.synchronize()
    for i in range(6):
        for c, st, o, w in zip(cases, streams, outs, ws):
            c.call(paged, out=o[i], workspace=w, stream=st)
    torch.cuda.synchronize()
    assert all(torch.equal(x, w) for o, w in zip(outs, want) for x in o) and K.status() == 0


def test_append_then_attention_without_a_pause(paged, K):
    """Steps back to back on one stream: each attention sees the keys that the append before it stored."""
    rows, nq, nkv, ps, steps = 5, 16, 4, 16, 40
    pool = paged.KVPool.zeros(rows * 4 + 20, nkv, ps, torch.float32)
    pre = torch.arange(20, dtype=torch.int32, device="cuda")
    pool.k[:20].normal_()
    pool.v[:20].normal_()
    table = torch.arange(20, 20 + rows * 4, dtype=torch.int32, device="cuda").view(rows, 4)
    rope = rope_table(1000)
    g = torch.Generator(device="cuda").manual_seed(1)
    qkv = torch.randn(steps, rows, (nq + 2 * nkv) * HD, generator=g, device="cuda")
    out = torch.empty(steps, rows, nq * HD, device="cuda")
    ws = paged.attention_workspace(rows, nq, nkv, 300, torch.float32)
    q = torch.empty(steps, rows, nq * HD, device="cuda")
    pos = torch.arange(steps, dtype=torch.int32, device="cuda")[:, None].expand(steps, rows).contiguous()
    slots = (table[:, (torch.arange(steps, device="cuda") // ps).long()].t() * ps + pos % ps).int().contiguous()
    lens = (pos + 1).contiguous()
    torch.cuda.synchronize()
    for t in range(steps):
        paged.append_kv(qkv[t], pool, slots[t], pos[t], rope, nq, first=300, q_out=q[t])
        paged.attention(q[t], pool, table, lens[t], prefix_pages=pre, prefix_len=300, out=out[t], workspace=ws)
    torch.cuda.synchronize()
    assert K.status() == 0
    k = torch.cat([pool.k[:20].transpose(0, 1).reshape(nkv, -1, HD)[:, :300][None].expand(rows, -1, -1, -1),
                   pool.k[table.long()].transpose(1, 2).reshape(rows, nkv, -1, HD)], 2).double()
    v = torch.cat([pool.v[:20].transpose(0, 1).reshape(nkv, -1, HD)[:, :300][None].expand(rows, -1, -1, -1),
                   pool.v[table.long()].transpose(1, 2).reshape(rows, nkv, -1, HD)], 2).double()
    for t in (0, 1, 15, 16, 39):
        p = torch.softmax(torch.einsum("bhgd,bhtd->bhgt", q[t].double().view(rows, nkv, nq // nkv, HD),
                                       k[:, :, :301 + t]) / math.sqrt(HD), -1)
        want = torch.einsum("bhgt,bhtd->bhgd", p, v[:, :, :301 + t]).reshape(rows, -1)
        mag = torch.einsum("bhgt,bhtd->bhgd", p, v[:, :, :301 + t].abs()).reshape(rows, -1)
        assert bool(((out[t].double() - want).abs() <= 1e-4 * mag).all())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attention_sharp_and_flat_scores(paged, K, dtype):
    """One key far above the rest (weights near 1 and near 0), then nearly equal scores, then scores of thousands."""
    for scale, tol in ((0.01, 1e-4), (4.0, 1e-3)):
        # a score's error grows with its terms: q.k terms sum to scale^2 * 7.3 on average, at most about four times that;
        # 2^-20 of it bounds each weight's relative error, below 1e-3 at scale 4
        c = Case(paged, 6, 16, 4, 300, [0, 1, 50, 200, 333, 16], 16, DTYPES[dtype], seed=3, scale=scale)
        c.check(c.call(paged), tol=tol, rms=tol / 10)
    c = Case(paged, 4, 8, 2, 100, [10, 20, 30, 0], 16, DTYPES[dtype], seed=4)
    c.q.mul_(300.0)  # the largest score alone counts; ties are not drawn
    want, _ = c.oracle()
    got = c.call(paged)
    assert bool(torch.isfinite(got).all())
    # weights e^(s - m) with scores of some thousands: fp32 scores are good to 2^-20 of 2^13
    assert float((got.double() - want).abs().max()) <= 0.05
    torch.cuda.synchronize()
    assert K.status() == 0


def test_attention_strides_stream_and_default_buffers(paged, K):
    c = Case(paged, 5, 16, 4, 40, [3, 0, 90, 17, 64], 16, torch.float16, seed=9)
    base = c.call(paged)
    wide_q = torch.full((5, 16 * HD + 4), 7.0, device="cuda")
    wide_q[:, :16 * HD] = c.q
    wide_o = torch.full((5, 16 * HD + 8), 7.0, device="cuda")
    wide_t = torch.full((5, c.table.shape[1] + 3), 99999, dtype=torch.int32, device="cuda")
    wide_t[:, :c.table.shape[1]] = c.table
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    paged.attention(wide_q[:, :16 * HD], c.pool, wide_t[:, :c.table.shape[1]], c.lens, prefix_pages=c.pre,
                    prefix_len=40, out=wide_o[:, :16 * HD], stream=side)
    side.synchronize()
    assert torch.equal(wide_o[:, :16 * HD], base) and bool((wide_o[:, 16 * HD:] == 7.0).all())
    # one list for all rows, each its own length: the rows of a block of positions of one sequence
    one = Case(paged, 1, 16, 4, 0, [90], 16, torch.float16, seed=10)
    q = torch.randn(6, 16 * HD, device="cuda")
    lens = [1, 16, 17, 50, 89, 90]
    got = paged.attention(q, one.pool, one.table[0], ints(lens))
    for j, n in enumerate(lens):
        one.q, one.lens_host = q[j:j + 1], [n]
        one.check(got[j:j + 1])
    assert K.status() == 0


def test_attention_lengths_are_clamped_and_bad_pages_left_out(paged, K):
    c = Case(paged, 3, 8, 2, 0, [64, 20, 33], 16, torch.float16, seed=11, slack=0)
    c.lens.copy_(ints([1000, -5, 33]))  # past the table's 4 pages; negative
    c.lens_host = [64, 0, 33]
    c.check(c.call(paged))
    assert K.status() == 0
    c.table[2, 1] = c.pool.n_pages  # keys 16 .. 31 of row 2 are left out
    got = c.call(paged)
    torch.cuda.synchronize()
    assert K.status() == 4
    keep = c.own_ids[2]
    c.pool.k[keep[1]] = c.pool.k[keep[2]]  # the oracle: page 1 holds page 2's one key, then nothing
    c.pool.v[keep[1]] = c.pool.v[keep[2]]
    c.own_ids[2], c.lens_host[2] = [keep[0], keep[1]], 17
    c.check(got)


@pytest.mark.parametrize("prefix", [700, 2500])
def test_attention_is_the_same_when_repeated_and_captured(paged, K, prefix):
    c = Case(paged, 9, 32, 4, prefix, [0, 9, 100, 1000, 64, 65, 3, 2, 1], 16, torch.bfloat16, seed=12)
    out = torch.empty(9, 32 * HD, device="cuda")
    ws = paged.attention_workspace(9, 32, 4, prefix, torch.bfloat16)
    first = c.call(paged, out=out, workspace=ws).clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        c.call(paged, out=out, workspace=ws)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, first)  # no result depends on the order in which CTAs finish
    c.lens.copy_(ints([5, 9, 100, 999, 64, 65, 3, 0, 1]))  # the captured call reads the lengths of its replay
    c.own_ids[0], c.lens_host = c.own_ids[1], [5, 9, 100, 999, 64, 65, 3, 0, 1]
    c.table[0, 0] = c.own_ids[1][0]
    graph.replay()
    torch.cuda.synchronize()
    c.check(out)
    assert K.status() == 0


def test_attention_offsets_past_32_bits(paged, K):
    """Keys and values beyond 2^31 elements from the pool's start."""
    nkv, ps = 8, 256
    pages = (1 << 31) // (nkv * ps * HD) + 3
    k = torch.zeros(pages, nkv, ps, HD, dtype=torch.float16, device="cuda")
    v = torch.zeros(pages, nkv, ps, HD, dtype=torch.float16, device="cuda")
    last = pages - 1
    k[last].normal_()
    v[last].normal_()
    k[last - 1].normal_()
    v[last - 1].normal_()
    c = Case(paged, 1, 8, nkv, 200, [100], ps, torch.float16, seed=1)
    c.pool = paged.KVPool(k, v)
    c.pre_ids, c.own_ids = [last - 1], [[last]]
    c.pre, c.table[0, 0] = ints([last - 1]), last
    c.check(c.call(paged))
    slot = last * ps + 255
    paged.append_kv(torch.ones(1, 3 * nkv * HD, device="cuda"), c.pool, ints([slot]), ints([0]), rope_table(2), nkv)
    torch.cuda.synchronize()
    assert bool((c.pool.v[last, :, 255] == 1).all()) and K.status() == 0


@pytest.mark.parametrize("bad", ["dtype", "heads", "prefix", "pages", "table", "lens", "out", "workspace", "device"])
def test_attention_wrapper_refuses(paged, K, bad):
    c = Case(paged, 2, 8, 2, 20, [5, 6], 16, torch.float16)
    q, table, lens, pre, n, kw = c.q, c.table, c.lens, c.pre, 20, {}
    if bad == "dtype":
        q = q.half()
    elif bad == "heads":
        q = q[:, :7 * HD]
    elif bad == "prefix":
        pre = None
    elif bad == "pages":
        n = 33
    elif bad == "table":
        table = table.long()
    elif bad == "lens":
        lens = lens[:1]
    elif bad == "out":
        kw["out"] = torch.empty(2, 4 * HD, device="cuda")
    elif bad == "workspace":
        kw["workspace"] = torch.empty(16, dtype=torch.uint8, device="cuda")
    else:
        lens = lens.cpu()
    with pytest.raises(ValueError):
        paged.attention(q, c.pool, table, lens, prefix_pages=pre, prefix_len=n, **kw)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("rows,nq,nkv,prefix,ps", [
    (16, 32, 4, 5000, 16), (8, 48, 6, 4609, 64), (16, 8, 1, 9001, 16), (7, 64, 8, 4100, 32), (16, 32, 4, 9217, 128)])
def test_attention_prefix_parts(paged, K, dtype, rows, nq, nkv, prefix, ps):
    """Prefixes cut into many parts, on half the SMs or on all, beside own keys of any length."""
    for lens in ([0] * rows, [(61 * j) % 701 for j in range(rows)]):
        c = Case(paged, rows, nq, nkv, prefix, lens, ps, DTYPES[dtype], seed=prefix + nkv)
        got = c.call(paged)
        torch.cuda.synchronize()
        assert K.status() == 0
        c.check(got)


@pytest.mark.parametrize("dtype,rows,nq,nkv,prefix", [
    ("f32", 1, 16, 8, 0), ("f32", 16, 16, 8, 300), ("f32", 5, 32, 2, 40), ("f16", 16, 32, 4, 0), ("bf16", 9, 32, 4, 700),
    ("f16", 16, 32, 4, 2100)])
def test_steps_without_a_pause(paged, K, dtype, rows, nq, nkv, prefix):
    """Tables, append and attention back to back, each step's lengths made on the device by the step before: the
    same as with a synchronisation behind every call."""
    ps, steps = 16, 50
    g = torch.Generator(device="cuda").manual_seed(rows)
    qkv = torch.randn(steps, rows, (nq + 2 * nkv) * HD, generator=g, device="cuda")
    fresh = (torch.rand(steps, rows, generator=g, device="cuda") < 0.8).to(torch.int32)
    rope, shared = rope_table(prefix + steps), pages_of(prefix, ps)
    width = pages_of(steps, ps)
    k0 = torch.randn(2, shared + rows * width, nkv, ps, HD, generator=g, device="cuda").to(DTYPES[dtype])
    ids = torch.arange(shared + rows * width, dtype=torch.int32, device="cuda")
    runs = []
    for pause in (True, False):
        pool = paged.KVPool(k0[0].clone(), k0[1].clone())
        two = [paged.TokenSlots.empty(rows, row_stride=1) for _ in range(2)]
        table, used = torch.full((rows, width), -1, dtype=torch.int32, device="cuda"), ints([shared])
        ws = paged.attention_workspace(rows, nq, nkv, prefix, DTYPES[dtype])
        q, out = torch.zeros(steps, rows, nq * HD, device="cuda"), torch.empty(steps, rows, nq * HD, device="cuda")
        rest = torch.cuda.synchronize if pause else (lambda: None)
        torch.cuda.synchronize()
        for t in range(steps):
            was, now = two[t % 2], two[(t + 1) % 2]
            paged.page_tables(was.kv_lens, fresh[t], ps, ids, used, table, now)
            rest()
            paged.append_kv(qkv[t], pool, now.slots, now.positions, rope, nq, first=prefix, q_out=q[t])
            rest()
            paged.attention(q[t], pool, table, now.kv_lens, prefix_pages=ids, prefix_len=prefix, out=out[t], workspace=ws)
            rest()
        torch.cuda.synchronize()
        runs.append((out, pool.k, pool.v, table, two[steps % 2].kv_lens))
    assert K.status() == 0
    assert torch.equal(runs[0][4], fresh.sum(0).int())
    for a, b in zip(*runs):
        assert torch.equal(a, b)
