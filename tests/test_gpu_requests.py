"""Forked requests, page copies and released pages on a B200, against host loops."""
from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

HD = 128


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
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def pages_of(n, ps):
    return -(-n // ps)


def host_fork(parents, lens, ps, free, used, table, shared):
    lens, table, shared, copies, ok, asked = list(lens), table.copy(), shared.copy(), [[], []], True, 0
    held = list(lens)
    for i, p in enumerate(parents):
        src = dst = -1
        if p >= 0:
            fine = p < len(lens) and parents[p] < 0 and held[i] == 0 and 0 <= held[p] <= table.shape[1] * ps
            part = fine and held[p] % ps > 0
            if fine and part and used + asked >= len(free):
                fine = False
            asked += part
            ok = ok and fine
            if fine:
                lens[i], full = held[p], held[p] // ps
                table[i, :full] = table[p, :full]
                np.add.at(shared, table[p, :full], 1)
                if part:
                    src, dst = table[p, full], free[used + asked - 1]
                    table[i, full] = dst
        copies[0].append(src)
        copies[1].append(dst)
    return lens, table, shared, np.array(copies), min(used + asked, len(free)), ok


def host_release(lens, keep, ps, free, used, table, shared):
    lens, free, shared, freed, ok = list(lens), free.copy(), shared.copy(), [], True
    gone = set()
    for i, n in enumerate(lens):
        if n < 0 or n > table.shape[1] * ps:
            ok = False
            continue
        lens[i] = min(max(keep[i], 0), n)
        for c in range(pages_of(lens[i], ps), pages_of(n, ps)):
            page = table[i, c]
            if page < 0 or page >= len(shared) or page in gone:
                ok = False
            elif shared[page] == 0:
                freed.append(page)
                gone.add(page)
            else:
                shared[page] -= 1
    at = used - len(freed)
    for p in sorted(freed):
        if 0 <= at < len(free):
            free[at] = p
        at += 1
    ok = ok and len(freed) <= used
    return lens, free, shared, max(used - len(freed), 0), ok


def state(rng, lens, ps, width, spare, share=1):
    """Tables of requests, `share` neighbours with common first pages; counts and the free list."""
    n = len(lens)
    need = sum(pages_of(max(x, 0), ps) for x in lens)
    ids = rng.permutation(need + spare).astype(np.int64)
    table, shared, used = np.full((n, width), -1, dtype=np.int64), np.zeros(need + spare, dtype=np.int64), 0
    for a in range(0, n, share):
        group = range(a, min(a + share, n))
        common = min(max(lens[i], 0) // ps for i in group) // 2 if len(group) > 1 else 0
        head = ids[used:used + common]
        used += common
        shared[head] = len(group) - 1
        for i in group:
            p = pages_of(max(lens[i], 0), ps)
            table[i, :common] = head
            table[i, common:p] = ids[used:used + p - common]
            used += p - common
    return table, shared, ids, used


def run_fork(paged, K, parents, lens, ps, table, shared, free, used, alias=False):
    want = host_fork(parents, lens, ps, free, used, table, shared)
    n, width = table.shape
    big = torch.full((n, width + 2), -7, dtype=torch.int32, device="cuda")
    big[:, :width] = ints(table)
    d_lens, d_used, d_shared = ints(lens), ints([used]), ints(shared)
    kw = {} if alias else dict(lens_out=torch.full_like(d_lens, -9), used_out=ints([-9]),
                               shared_out=torch.full_like(d_shared, -9), copies=torch.full((2, n), -9, dtype=torch.int32, device="cuda"))
    copies = paged.fork_requests(ints(parents), d_lens, ps, ints(free), d_used, big[:, :width], d_shared, **kw)
    torch.cuda.synchronize()
    status = K.status()
    assert (kw.get("lens_out", d_lens)).tolist() == want[0]
    assert np.array_equal(big[:, :width].cpu().numpy(), want[1]) and bool((big[:, width:] == -7).all())
    assert np.array_equal(kw.get("shared_out", d_shared).cpu().numpy(), want[2])
    assert np.array_equal(copies.cpu().numpy(), want[3])
    assert int(kw.get("used_out", d_used)) == want[4] and status == (0 if want[5] else 4)
    if not alias:
        assert d_lens.tolist() == list(lens) and int(d_used) == used and np.array_equal(d_shared.cpu().numpy(), shared)
    return want


def run_release(paged, K, lens, keep, ps, table, shared, free, used, alias=False):
    want = host_release(lens, keep, ps, free, used, table, shared)
    n, width = table.shape
    big = torch.full((n, width + 2), 3, dtype=torch.int32, device="cuda")
    big[:, :width] = ints(table)
    d_lens, d_used, d_shared, d_free = ints(lens), ints([used]), ints(shared), ints(free)
    kw = {} if alias else dict(lens_out=torch.full_like(d_lens, -9), used_out=ints([-9]),
                               shared_out=torch.full_like(d_shared, -9))
    paged.release_pages(d_lens, ints(keep), ps, d_free, d_used, big[:, :width], d_shared, **kw)
    torch.cuda.synchronize()
    status = K.status()
    assert (kw.get("lens_out", d_lens)).tolist() == want[0]
    assert np.array_equal(d_free.cpu().numpy(), want[1])
    assert np.array_equal(kw.get("shared_out", d_shared).cpu().numpy(), want[2])
    assert int(kw.get("used_out", d_used)) == want[3] and status == (0 if want[4] else 4)
    assert np.array_equal(big[:, :width].cpu().numpy(), table)
    return want


@pytest.mark.parametrize("n,parents,held,ps,spare", [
    (2, 1, 40, 16, 5), (2, 1, 32, 16, 0), (16, 1, 1003, 16, 20), (128, 16, 700, 64, 200), (9, 4, 5, 128, 9),
    (4080, 100, 90, 16, 4000), (33, 3, 20000, 16, 40)])
@pytest.mark.parametrize("alias", [False, True])
def test_fork_matches_the_host_loop(paged, K, n, parents, held, ps, spare, alias):
    rng = np.random.default_rng(n + held)
    lens = [held] + rng.integers(0, held + 1, parents - 1).tolist() + [0] * (n - parents)
    of = [-1] * parents + [int(x) for x in rng.integers(-1, parents, n - parents)]
    table, shared, free, used = state(rng, lens, ps, pages_of(held, ps) + 1, spare)
    run_fork(paged, K, of, lens, ps, table, shared, free, used, alias)


def test_fork_requests_that_cannot_be_served(paged, K):
    rng = np.random.default_rng(1)
    lens = [40, 33, 0, 0, 0, 7, 0, 0, 0]
    table, shared, free, used = state(rng, lens, 16, 4, 6)
    # itself, a row past the end, a parent that is a child, a row that holds tokens, and two that are fine
    want = run_fork(paged, K, [-1, -1, 2, 9, 0, 0, 4, 1, 2 ** 31 - 1], lens, 16, table, shared, free, used)
    assert not want[5] and want[0] == [40, 33, 0, 0, 40, 7, 0, 33, 0]
    # the free list runs out: later rows that need a page are left out, others not
    lens = [40, 32, 0, 0, 0, 0]
    table, shared, free, used = state(rng, lens, 16, 3, 1)
    want = run_fork(paged, K, [-1, -1, 0, 0, 1, 0], lens, 16, table, shared, free, used, alias=True)
    assert not want[5] and want[0] == [40, 32, 40, 0, 32, 0]
    # parents longer than their row, or of negative length; a parent with nothing
    table[:] = 0
    run_fork(paged, K, [-1, -1, -1, 0, 1, 2], [49, -1, 0, 0, 0, 0], 16, table, shared, free, used)
    # a count outside the list
    for bad in (-1, len(free) + 1):
        d = [ints(x) for x in ([-1, 0], [20, 0], free, [bad], shared)]
        t = torch.zeros(2, 2, dtype=torch.int32, device="cuda")
        copies = paged.fork_requests(d[0], d[1], 16, d[2], d[3], t, d[4])
        torch.cuda.synchronize()
        assert K.status() == 4 and int(d[3]) == bad and bool((copies == -1).all()) and d[1].tolist() == [20, 0]


def test_fork_pages_outside_the_pool(paged, K):
    lens, table = ints([40, 0, 0]), ints([[5, -1, 9], [-1] * 3, [-1] * 3])
    shared, free, used = torch.zeros(12, dtype=torch.int32, device="cuda"), ints([0, 99, 3]), ints([1])
    copies = paged.fork_requests(ints([-1, 0, 0]), lens, 16, free, used, table, shared)
    torch.cuda.synchronize()
    assert K.status() == 4
    assert shared.tolist() == [2 if p == 5 else 0 for p in range(12)]
    assert copies.tolist() == [[-1, -1, 9], [-1, -1, 3]] and lens.tolist() == [40, 40, 40]


@pytest.mark.parametrize("n,held,back,ps,spare,share", [
    (1, 1, 1, 16, 0, 1), (16, 2000, 4, 16, 4000, 1), (128, 4000, 4000, 16, 30000, 4), (7, 300, 200, 128, 3, 2),
    (4080, 60, 60, 16, 100, 5), (3, 100000, 100000, 16, 10, 1), (5, 40, 0, 16, 2, 5)])
@pytest.mark.parametrize("alias", [False, True])
def test_release_matches_the_host_loop(paged, K, n, held, back, ps, spare, share, alias):
    rng = np.random.default_rng(n + held)
    lens = [held] + rng.integers(0, held + 1, n - 1).tolist()
    keep = [x - int(rng.integers(0, back + 1)) for x in lens]  # some below zero: all goes
    if n > 2:
        keep[1] = lens[1] + 5  # nothing goes
        keep[2] = 0
    table, shared, free, used = state(rng, lens, ps, pages_of(held, ps) + 1, spare, share)
    run_release(paged, K, lens, keep, ps, table, shared, free, used, alias)


def test_release_all_holders_and_nothing(paged, K):
    rng = np.random.default_rng(3)
    lens = [100] * 6
    table, shared, free, used = state(rng, lens, 16, 8, 11, 6)
    want = run_release(paged, K, lens, [0] * 6, 16, table, shared, free, used)
    assert want[3] == 0 and sorted(want[1].tolist()) == sorted(free.tolist()) and not want[2].any()
    run_release(paged, K, lens, lens, 16, table, shared, free, used, alias=True)


def test_release_what_is_not_held(paged, K):
    """Ids outside the pool, a page released twice, lengths outside the row, more pages than were taken."""
    rng = np.random.default_rng(4)
    lens = [64, 64, -3, 65, 20]
    table, shared, free, used = state(rng, [64, 64, 0, 20, 20], 16, 4, 5)
    table[0, 1], table[1, 2], table[1, 3] = -1, len(shared), table[1, 0]
    want = run_release(paged, K, lens, [0] * 5, 16, table, shared, free, used)
    assert not want[4] and want[0] == [0, 0, -3, 65, 0]
    table, shared, free, used = state(rng, [64, 64], 16, 4, 5)
    run_release(paged, K, [64, 64], [0, 0], 16, table, shared, free, 3)
    assert not host_release([64, 64], [0, 0], 16, free, 3, table, shared)[4]


def test_release_a_million_pages(paged, K):
    n = 1 << 20
    shared = torch.zeros(n, dtype=torch.int32, device="cuda")
    for pages in ([n - 1, 0, 31, 32, n // 2], [n // 8 * j for j in range(8)]):
        table, free = ints([pages]), torch.full((n,), -5, dtype=torch.int32, device="cuda")
        used = ints([n])
        paged.release_pages(ints([16 * len(pages)]), ints([0]), 16, free, used, table, shared)
        torch.cuda.synchronize()
        assert K.status() == 0 and int(used) == n - len(pages)
        assert free[-len(pages):].tolist() == sorted(pages) and bool((free[:-len(pages)] == -5).all())
    with pytest.raises(ValueError):
        paged.release_pages(ints([16]), ints([0]), 16, free, used, table,
                            torch.zeros(n + 1, dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("dtype,nkv,ps,layers,n", [
    (torch.float32, 8, 16, 3, 20), (torch.float16, 1, 16, 70, 5), (torch.bfloat16, 3, 256, 2, 1),
    (torch.float16, 4, 64, 130, 40)])
def test_copy_pages(paged, K, dtype, nkv, ps, layers, n):
    g = torch.Generator(device="cuda").manual_seed(n)
    pages = 2 * n + 5
    k, v = (torch.randn(layers, pages, nkv, ps, HD, generator=g, device="cuda").to(dtype) for _ in range(2))
    pools = [paged.KVPool(a, b) for a, b in zip(k, v)]
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    copies = order[:2 * n].view(2, n).clone()
    copies[0, n // 2] = copies[0, 0]  # one source of two copies
    if n > 4:
        copies[1, 3] = -1
        copies[0, 4] = -1
    want = [x.clone() for x in (k, v)]
    for s, d in copies.t().tolist():
        if s >= 0 and d >= 0:
            for w in want:
                w[:, d] = w[:, s]
    paged.copy_pages(pools, copies)
    torch.cuda.synchronize()
    assert K.status() == 0 and torch.equal(k, want[0]) and torch.equal(v, want[1])
    bad = copies.clone()
    bad[0, 0], bad[1, n - 1] = pages, -2
    if n > 1:
        paged.copy_pages(pools, bad)
        torch.cuda.synchronize()
        assert K.status() == 4 and torch.equal(k, want[0]) and torch.equal(v, want[1])
    paged.copy_pages(pools, copies[:, :0])
    paged.copy_pages([], copies)
    with pytest.raises(ValueError, match="one shape"):
        paged.copy_pages(pools + [paged.KVPool.zeros(3, nkv, ps, dtype)], copies)
    with pytest.raises(ValueError):
        paged.copy_pages(pools, copies.long())


def test_copy_pages_past_32_bits(paged, K):
    nkv, ps = 8, 256
    pages = (1 << 31) // (nkv * ps * HD) + 3
    pool = paged.KVPool.zeros(pages, nkv, ps, torch.float16)
    pool.k[1].normal_()
    pool.v[pages - 1].normal_()
    paged.copy_pages([pool], ints([[1, pages - 1], [pages - 2, 0]]))
    torch.cuda.synchronize()
    assert torch.equal(pool.k[1], pool.k[pages - 2]) and torch.equal(pool.v[0], pool.v[pages - 1]) and K.status() == 0


def test_steps_of_forks_and_releases_in_a_graph(paged, K):
    """Tables, fork and release replayed: what is taken comes back, no page is lost or held twice."""
    n, ps, width = 12, 16, 6
    rng = np.random.default_rng(0)
    total = n * width
    free, used, shared = ints(rng.permutation(total)), ints([0]), torch.zeros(total, dtype=torch.int32, device="cuda")
    table, lens = torch.full((n, width), -1, dtype=torch.int32, device="cuda"), ints([0] * n)
    new, parents, keep = ints([0] * n), ints([-1] * n), ints([0] * n)
    out = paged.TokenSlots.empty(n, row_stride=20)
    copies = torch.empty(2, n, dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        paged.release_pages(lens, keep, ps, free, used, table, shared)
        paged.fork_requests(parents, lens, ps, free, used, table, shared, copies=copies)
        paged.page_tables(lens, new, ps, free, used, table, out)
        lens.copy_(out.kv_lens)
    host = [[0] * n, np.full((n, width), -1, dtype=np.int64), np.zeros(total, dtype=np.int64), free.cpu().numpy().astype(np.int64), 0]
    for step in range(40):
        k = [0 if rng.random() < 0.3 else 10 ** 6 for _ in range(n)]
        if step % 3 == 0:  # drafts refused: not below a page that others hold
            k = [x if x == 0 else max(0, m - int(rng.integers(0, 3))) if m % ps > 3 else x for x, m in zip(k, host[0])]
        after = [min(x, m) for x, m in zip(k, host[0])]
        live = [i for i in range(n) if after[i] > 0]
        of = [int(rng.choice(live)) if live and after[i] == 0 and rng.random() < 0.5 else -1 for i in range(n)]
        lens_now, host[3], host[2], host[4], ok = host_release(host[0], k, ps, host[3], host[4], host[1], host[2])
        assert ok
        lens_now, host[1], host[2], want_copies, host[4], ok = host_fork(of, lens_now, ps, host[3], host[4], host[1], host[2])
        assert ok
        fresh = [int(rng.integers(0, 20)) if m + 20 <= width * ps else 0 for m in lens_now]
        for i in range(n):  # the block tables, on the host
            for c in range(pages_of(lens_now[i], ps), pages_of(lens_now[i] + fresh[i], ps)):
                host[1][i, c] = host[3][host[4]]
                host[4] += 1
        host[0] = [a + b for a, b in zip(lens_now, fresh)]
        keep.copy_(ints(k))
        parents.copy_(ints(of))
        new.copy_(ints(fresh))
        graph.replay()
        torch.cuda.synchronize()
        assert K.status() == 0 and lens.tolist() == host[0] and int(used) == host[4]
        assert np.array_equal(shared.cpu().numpy(), host[2]) and np.array_equal(copies.cpu().numpy(), want_copies)
        for i in range(n):
            assert table[i, :pages_of(host[0][i], ps)].tolist() == host[1][i, :pages_of(host[0][i], ps)].tolist()
        held = np.bincount(np.concatenate([host[1][i, :pages_of(host[0][i], ps)] for i in range(n)] + [np.zeros(0, int)]).astype(int), minlength=total)
        taken = held > 0
        assert np.array_equal(host[2][taken], held[taken] - 1) and taken.sum() == host[4]
        assert sorted(free[host[4]:].tolist()) == np.flatnonzero(~taken).tolist()


@pytest.mark.parametrize("bad", ["parents", "copies", "shared", "used", "table", "page", "device", "lens_out"])
def test_fork_and_release_refuse(paged, K, bad):
    n = 4
    parents, lens, keep = ints([-1] * n), ints([0] * n), ints([0] * n)
    free, used, table = ints(range(20)), ints([0]), torch.zeros(n, 3, dtype=torch.int32, device="cuda")
    shared, ps, kw = torch.zeros(20, dtype=torch.int32, device="cuda"), 16, {}
    both = bad not in ("parents", "copies", "lens_out")
    if bad == "parents":
        parents = parents[:3]
    elif bad == "copies":
        kw["copies"] = ints([[0] * n])
    elif bad == "shared":
        shared = shared.long()
    elif bad == "used":
        used = ints([0, 0])
    elif bad == "table":
        table = table[:3]
    elif bad == "page":
        ps = 24
    elif bad == "device":
        shared = shared.cpu()
    else:
        kw["lens_out"] = parents
    with pytest.raises(ValueError):
        paged.fork_requests(parents, lens, ps, free, used, table, shared, **kw)
    if both:
        with pytest.raises(ValueError):
            paged.release_pages(lens, keep, ps, free, used, table, shared)
    torch.cuda.synchronize()
    assert K.status() == 0


def test_copy_pages_leaves_out_bad_pages_alone(paged, K):
    """Every page of its own content: pages outside the pool are neither copied nor redirected, the others are copied."""
    pages, layers = 20, 3
    g = torch.Generator(device="cuda").manual_seed(5)
    k, v = (torch.randn(layers, pages, 2, 16, HD, generator=g, device="cuda").half() for _ in range(2))
    pools = [paged.KVPool(a, b) for a, b in zip(k, v)]
    copies = [[0, pages, 2, -2, 4, 5, 2 ** 31 - 1, 7, -1], [10, 11, pages, 13, -2 ** 31, 15, 16, 17, 18]]
    want = [x.clone() for x in (k, v)]
    for s, d in zip(*copies):
        if 0 <= s < pages and 0 <= d < pages:
            for w in want:
                w[:, d] = w[:, s]
    paged.copy_pages(pools, ints(copies))
    torch.cuda.synchronize()
    assert K.status() == 4 and torch.equal(k, want[0]) and torch.equal(v, want[1])
    assert not torch.equal(want[0][:, 10], want[0][:, 11]) and torch.equal(k[:, 17], k[:, 7])
