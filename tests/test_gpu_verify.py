"""Token distributions and the verification of drafts on a B200, against the definitions in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def S(cuda_device):
    from pyrite_b200.kernels import cuda, sampling
    cuda.status()
    return sampling


def cuda(x, d=torch.float32):
    return None if x is None else torch.as_tensor(np.asarray(x)).to(d).cuda()


# ---- token_probs -----------------------------------------------------------------------------
def distribution(row, temp, k, p, mp):
    """(probabilities, sharp): sharp is false where a border lies within the kernel's error of a sum."""
    row = np.where(np.isnan(row), -np.inf, row.astype(np.float64))
    out = np.zeros(row.size)
    order = np.lexsort((np.arange(row.size), -row))
    top = row[order[0]]
    if top == -np.inf:
        return out, True
    if not temp > 0:
        out[order[0]] = 1.0
        return out, True
    r = row[order]
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(r == top, 1.0, np.exp((r - top) / float(temp)))
    err, sharp = row.size * 2.0 ** -42 + 1e-13, True
    n = row.size if k <= 0 else min(k, row.size)
    cum = np.cumsum(w[:n])
    if p < 1:
        target = max(float(p), 0.0) * cum[-1]
        n = min(int(np.searchsorted(cum, target, side="left")), n - 1) + 1
        sharp = np.abs(cum - target).min() > err * 4 or target == 0.0
    if mp > 0:
        n = min(n, max(1, int((w >= min(float(mp), 1.0)).sum())))
    out[order[:n]] = w[:n] / w[:n].sum()
    return out, sharp


def check_probs(S, logits, temp, k=None, p=None, mp=None, ld=None, sharp_share=0.9):
    rows, n = logits.shape
    dev = cuda(logits)
    if ld:
        wide = torch.full((rows, ld), 1e30, device="cuda")
        wide[:, :n] = dev
        dev = wide[:, :n]
        out = torch.full((rows, ld + 1), -7.0, device="cuda")
        got = S.token_probs(dev, cuda(temp), top_k=cuda(k, torch.int32), top_p=cuda(p), min_p=cuda(mp), out=out[:, 1:n + 1])
        assert bool((out[:, 0] == -7.0).all()) and bool((out[:, n + 1:] == -7.0).all())
    else:
        got = S.token_probs(dev, cuda(temp), top_k=cuda(k, torch.int32), top_p=cuda(p), min_p=cuda(mp))
    got, host, sharp_rows = got.double().cpu().numpy(), dev.cpu().numpy(), 0
    at = lambda x, i, off: off if x is None else np.float32(x[i])  # noqa: E731
    for j in range(rows):
        want, sharp = distribution(host[j], np.float32(temp[j]), 0 if k is None else int(k[j]), at(p, j, np.float32(1)),
                                   at(mp, j, np.float32(0)))
        if not sharp:
            continue
        sharp_rows += 1
        # half a step of fp32 (or of its subnormals), and the kept mass: n units of 2^-42 of the largest weight at worst
        tol = want * (2.0 ** -24 + n * 2.0 ** -42 + 1e-12) + 2.0 ** -150
        assert (np.abs(got[j] - want) <= tol).all(), (j, np.abs(got[j] - want).max())
    assert sharp_rows >= sharp_share * rows


@pytest.mark.parametrize("n", [1, 2, 3, 31, 33, 128, 1000, 1025, 4097, 32000, 50257, 128256, 151936])
def test_probs_settings_over_vocabularies(S, n):
    rng = np.random.default_rng(n)
    rows = 24
    logits = rng.normal(0, 2.5, (rows, n)).astype(np.float32)
    logits[:, rng.integers(0, n, 5)] += rng.uniform(0, 9, (rows, 5)).astype(np.float32)
    temp = rng.choice([0.0, 0.3, 0.8, 1.0, 1.7, 5.0], rows)
    k = rng.choice([0, 1, 2, 40, 1000, 5000, n, n + 7], rows)
    p = rng.choice([0.0, 0.1, 0.5, 0.9, 0.99, 0.9999, 1.0, 2.0], rows)
    mp = rng.choice([0.0, 0.0, 1e-6, 0.02, 0.3, 1.0, 1.5], rows)
    check_probs(S, logits, temp, k, p, mp, sharp_share=0.8)
    check_probs(S, logits, np.full(rows, 1.0))  # every filter off
    check_probs(S, logits, temp, k=k, ld=n + 3)
    check_probs(S, logits, temp, p=p, sharp_share=0.8)
    check_probs(S, logits, temp, mp=mp)


@pytest.mark.parametrize("n", [7, 4096, 151936])
def test_probs_ties_and_special_rows(S, n):
    rng = np.random.default_rng(n + 1)
    rows = 12
    flat = np.zeros((rows, n), dtype=np.float32)
    flat[1::2] = -0.0
    k = [min(n, x) for x in (1, 2, 5, n // 2 + 1, n - 1, n, 3, n // 3 + 1, 1, 2, 4, n)]
    check_probs(S, flat, np.full(rows, 0.7), k=k)
    coarse = rng.integers(0, 4, (rows, n)).astype(np.float32)  # long runs of one value
    check_probs(S, coarse, np.full(rows, 1.0), k=k)
    check_probs(S, coarse, np.full(rows, 0.5), p=rng.uniform(0.2, 0.95, rows), sharp_share=0.5)
    odd = rng.normal(0, 3, (rows, n)).astype(np.float32)
    odd[0] = -np.inf
    odd[1] = np.nan
    odd[2, : n // 2] = np.nan
    odd[3, ::2] = -np.inf
    odd[4, 3:6] = np.inf
    odd[5] = -np.inf
    odd[5, n - 1] = -1e30
    odd[6] *= 1e30
    odd[7] = np.float32(-3.4028235e38)
    odd[8, 1:] = np.float32(-3.4028235e38)
    for temp in (np.full(rows, 1.0), np.zeros(rows), np.full(rows, np.nan), np.full(rows, 30.0)):
        check_probs(S, odd, temp)
        check_probs(S, odd, temp, k=[3] * rows)
        check_probs(S, odd, temp, mp=[0.5] * rows)


def test_probs_agree_with_sampling(S):
    """The probability that sampling reports is the token's in the distribution, which sums to 1."""
    g = torch.Generator(device="cuda").manual_seed(0)
    rows, n = 40, 32000
    logits = torch.randn(rows, n, generator=g, device="cuda") * 3
    temp, u = torch.rand(rows, generator=g, device="cuda") + 0.3, torch.rand(rows, generator=g, device="cuda")
    top_p, top_k = torch.rand(rows, generator=g, device="cuda"), torch.randint(0, 3000, (rows,), generator=g, device="cuda").int()
    ids, share = S.sample_rows(logits, u, temp, top_k=top_k, top_p=top_p)
    probs = S.token_probs(logits, temp, top_k=top_k, top_p=top_p)
    # both are one rounding of the same quotient
    assert torch.equal(probs.gather(1, ids.long()[:, None])[:, 0], share) or bool(
        ((probs.gather(1, ids.long()[:, None])[:, 0] - share).abs() <= 2.0 ** -23 * share).all())
    assert bool(((probs.double().sum(-1) - 1).abs() <= n * 2.0 ** -42 + 2.0 ** -24).all())


@pytest.mark.parametrize("n", [(1 << 20) - 3, 1 << 20])
def test_probs_widest_rows(S, n):
    rng = np.random.default_rng(5)
    logits = rng.normal(0, 2, (3, n)).astype(np.float32)
    check_probs(S, logits, [1.0, 0.8, 1.0], k=[0, 7000, 0], p=[1.0, 1.0, 0.9], sharp_share=0.3)


def test_probs_refuse(S):
    x, t = torch.zeros(2, 8, device="cuda"), torch.ones(2, device="cuda")
    for bad in (dict(logits=x.half()), dict(logits=x[0]), dict(temperature=t[:1]), dict(top_k=t), dict(top_p=t.double()),
                dict(out=x), dict(out=torch.zeros(2, 7, device="cuda")), dict(min_p=t.cpu())):
        with pytest.raises(ValueError):
            S.token_probs(**{**dict(logits=x, temperature=t), **bad})


# ---- verify_drafts -----------------------------------------------------------------------------
def verify(p, x, starts, u, pick, q=None):
    p, q = (None if t is None else np.maximum(np.nan_to_num(t.astype(np.float64)), 0.0) for t in (p, q))
    out, counts, n = np.full(len(x), -9), [], p.shape[1]
    for i, a in enumerate(starts[:-1]):
        b = starts[i + 1]
        if b <= a:
            counts.append(0)
            continue
        out[a:b] = -1
        r = a
        while r < b - 1 and 0 <= x[r] < n and float(u[r]) * (1.0 if q is None else q[r, x[r]]) < p[r, x[r]]:
            out[r] = x[r]
            r += 1
        w = p[r].copy()
        if r < b - 1 and 0 <= x[r] < n:
            if q is None:
                w[x[r]] = 0.0
            else:
                w = np.maximum(w - q[r], 0.0)
            if w.sum() <= 0:
                w = p[r].copy()
        cum = np.cumsum(w)
        if not 0 < cum[-1] < np.inf:
            counts.append(r - a)
            continue
        at = min(int(np.searchsorted(cum, float(pick[i]) * cum[-1], side="right")), n - 1)
        out[r] = at
        counts.append(r - a + 1)
    return out, counts


def run_verify(S, p, x, starts, u, pick, q=None, wide=0):
    want, counts = verify(p, x, starts, u, pick, q)
    i32 = torch.int32
    dp, dq = cuda(p), cuda(q)
    if wide:
        store = torch.full((p.shape[0], p.shape[1] + wide), 5.0, device="cuda")
        store[:, 1:p.shape[1] + 1] = dp
        dp = store[:, 1:p.shape[1] + 1]
    out = torch.full((len(x),), -9, dtype=i32, device="cuda")
    got, number = S.verify_drafts(dp, cuda(x, i32), cuda(starts, i32), cuda(u), cuda(pick), draft_probs=dq, out=out)
    assert got is out and got.tolist() == want.tolist() and number.tolist() == counts
    tokens = cuda(x, i32)  # in place
    S.verify_drafts(dp, tokens, cuda(starts, i32), cuda(u), cuda(pick), draft_probs=dq, out=tokens, counts=number)
    own = torch.full((len(x),), -9, dtype=i32, device="cuda")
    for a, b in zip(starts[:-1], starts[1:]):
        own[a:b] = tokens[a:b]
    assert own.tolist() == want.tolist() and number.tolist() == counts
    return want, counts


def softmax(x):
    e = np.exp((x - x.max(-1, keepdims=True)).astype(np.float64))
    return (e / e.sum(-1, keepdims=True)).astype(np.float32)


@pytest.mark.parametrize("n", [1, 2, 5, 127, 2048, 2049, 32000, 128256, 151936])
@pytest.mark.parametrize("requests,drafts", [(1, 7), (16, 4), (70, 2), (3, 40)])
def test_verify_over_vocabularies(S, n, requests, drafts):
    if n * requests * drafts > 2e7:
        pytest.skip("covered by the smaller ones")
    rng = np.random.default_rng(n + requests)
    count = rng.integers(0, drafts + 2, requests)  # rows of a request: none, one (no draft), several
    count[0] = drafts + 1
    starts = [2] + (2 + np.cumsum(count)).tolist()
    rows = starts[-1] + 3
    logits = rng.normal(0, 2.5, (rows, n))
    logits[np.arange(rows), rng.integers(0, n, rows)] += 6
    p = softmax(logits)
    p[p < 1e-6] = 0.0
    q = softmax(logits + rng.normal(0, 0.8, (rows, n)))
    x = np.array([int(np.searchsorted(np.cumsum(row.astype(np.float64)), rng.random() * row.sum())) for row in q]).clip(0, n - 1)
    x[rng.random(rows) < 0.05] = rng.choice([-1, n, 2 ** 31 - 1])
    u, pick = rng.random(rows).astype(np.float32), rng.random(requests).astype(np.float32)
    run_verify(S, p, x, starts, u, pick, q)
    likely = np.where(rng.random(rows) < 0.8, p.argmax(-1), x)
    run_verify(S, p, likely, starts, u, pick, None, wide=3)


def test_verify_borders(S):
    """Equal distributions accept everything; u at exactly p / q refuses; nothing left falls back to p."""
    n, rows = 6, 5
    p = np.array([[0, 0.25, 0.5, 0.25, 0, 0]] * rows, dtype=np.float32)
    x = np.array([1, 2, 3, 1, 0])
    near = np.float32(1) - np.float32(2.0 ** -24)
    _, counts = run_verify(S, p, x, [0, rows], [near] * rows, [0.3], p.copy())
    assert counts == [rows]
    q = p.copy()
    q[1] = [0, 0, 1, 0, 0, 0]
    # u q = p exactly: not accepted; a step below: accepted
    assert run_verify(S, p, x, [0, rows], [0.0, 0.5, 0, 0, 0], [0.0], q)[1] == [2]
    assert run_verify(S, p, x, [0, rows], [0.0, np.nextafter(np.float32(0.5), np.float32(0)), 0, 0, 0], [0.0], q)[1] == [5]
    # a draft of probability 0 is refused even at u = 0; pick 0 and the largest random number
    z = np.array([0, 4, 5, 0, 0])
    assert run_verify(S, p, z, [0, 2, rows], [0.0] * rows, [0.0, near])[0].tolist() == [1, -1, 3, -1, -1]
    # p below q everywhere: the rest is empty, the token comes from p
    half = (p * np.float32(0.5)).astype(np.float32)
    assert run_verify(S, half, np.array([1, 1, 1, 1, 1]), [0, rows], [0.9] * rows, [0.5], p)[1] == [1]
    # a lookup that holds all probability but is refused, and rows of zeros, NaN and infinity
    one = np.zeros((rows, n), dtype=np.float32)
    one[:, 2] = 1.0
    one[2:, 2] = [0.0, np.nan, np.inf]
    assert run_verify(S, one[:4], np.full(4, 2), [0, 2, 3, 4], [1.0] * 4, [0.5, 0.5, 0.5])[1] == [1, 0, 0]
    got, counts = S.verify_drafts(cuda(one[4:]), cuda([2], torch.int32), cuda([0, 1], torch.int32), cuda([0.0]), cuda([0.5]))
    assert got.tolist() == [-1] and counts.tolist() == [0]


@pytest.mark.parametrize("draft", [False, True])
def test_verify_gives_the_targets_distribution(S, draft):
    """20000 requests of one draft: the first token's frequencies are p's, whatever q is."""
    rng = np.random.default_rng(7)
    n, count = 5, 20000
    p = np.array([0.4, 0.05, 0.3, 0.0, 0.25], dtype=np.float32)
    q = np.array([0.1, 0.5, 0.2, 0.15, 0.05], dtype=np.float32)
    x = np.zeros(2 * count, dtype=np.int64)
    x[::2] = rng.choice(n, count, p=(q / q.sum()).astype(np.float64) / (q / q.sum()).astype(np.float64).sum())
    tokens, counts = S.verify_drafts(cuda(np.tile(p, (2 * count, 1))), cuda(x, torch.int32),
                                     cuda(np.arange(count + 1) * 2, torch.int32), cuda(rng.random(2 * count)),
                                     cuda(rng.random(count)), draft_probs=cuda(np.tile(q, (2 * count, 1))) if draft else None)
    first = np.bincount(tokens[::2].cpu().numpy(), minlength=n) / count
    # five standard deviations of a share of 20000 draws
    assert (np.abs(first - p) <= 5 * np.sqrt(p * (1 - p) / count) + 1e-12).all()
    assert set(counts.tolist()) == {1, 2}


def test_verify_starts_outside_the_rows(S):
    p = np.tile(np.array([0.0, 0.5, 0.5], dtype=np.float32), (4, 1))
    i32 = torch.int32
    out = torch.full((4,), -9, dtype=i32, device="cuda")
    _, counts = S.verify_drafts(cuda(p), cuda([1, 1, 1, 1], i32), cuda([-5, 2, 1, 99], i32), cuda([0.0] * 4),
                                cuda([0.9, 0.9, 0.1]), out=out)
    torch.cuda.synchronize()
    assert counts.tolist() == [2, 0, 3]


def test_verify_on_a_stream_and_captured(S):
    rng = np.random.default_rng(3)
    rows, n = 12, 20000
    p, q = (softmax(rng.normal(0, 2, (rows, n))) for _ in range(2))
    args = [cuda(p), cuda(rng.integers(0, n, rows), torch.int32), cuda([0, 4, 5, 12], torch.int32), cuda(rng.random(rows)),
            cuda(rng.random(3))]
    kw = dict(draft_probs=cuda(q), out=torch.empty(rows, dtype=torch.int32, device="cuda"),
              counts=torch.empty(3, dtype=torch.int32, device="cuda"))
    want = [t.clone() for t in S.verify_drafts(*args, **kw)]
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    got = S.verify_drafts(*args, draft_probs=kw["draft_probs"], stream=side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    logits, temp = cuda(rng.normal(0, 2, (rows, n))), cuda([0.8] * rows)
    with torch.cuda.graph(graph):
        S.token_probs(logits, temp, out=args[0])
        S.verify_drafts(*args, **kw)
    for _ in range(3):
        logits.copy_(cuda(rng.normal(0, 2, (rows, n))))
        graph.replay()
        torch.cuda.synchronize()
        now = [t.clone() for t in (kw["out"], kw["counts"])]
        again = S.verify_drafts(S.token_probs(logits, temp), *args[1:], draft_probs=kw["draft_probs"])
        assert all(torch.equal(a, b) for a, b in zip(now, again))


def test_verify_refuses(S):
    i32 = torch.int32
    good = dict(probs=torch.zeros(4, 8, device="cuda"), draft_tokens=cuda([0] * 4, i32), starts=cuda([0, 4], i32),
                accept=torch.zeros(4, device="cuda"), pick=torch.zeros(1, device="cuda"))
    for bad in (dict(probs=good["probs"].double()), dict(draft_tokens=cuda([0] * 3, i32)), dict(starts=cuda([0], i32)),
                dict(accept=torch.zeros(3, device="cuda")), dict(pick=good["pick"].half()),
                dict(draft_probs=torch.zeros(4, 7, device="cuda")), dict(out=cuda([0] * 5, i32)),
                dict(counts=cuda([0], torch.int64)), dict(starts=cuda([0, 4], i32).cpu())):
        with pytest.raises(ValueError):
            S.verify_drafts(**{**good, **bad})


# ---- token_probs: temperatures, logits and filters at the end of their ranges ------------------
def uncut(row, temp, mp=0.0):
    """The definition without top-k and top-p, also for an infinite temperature: a logit that is not finite, or
    further below the largest than fp32's largest number, has no weight."""
    x = np.where(np.isnan(row), -np.inf, row.astype(np.float64))
    top = x.max()
    there = top - x <= np.finfo(np.float32).max
    w = np.where(there, np.exp(np.where(there, x - top, 0.0) / np.float64(temp)), 0.0)
    w[w < min(float(np.float32(mp)), 1.0)] = 0.0
    return w / w.sum()


@pytest.mark.parametrize("n", [5, 1000, 151936])
@pytest.mark.parametrize("temp", [np.inf, 3.4028234e38, 1e30, 2.0])
def test_probs_at_large_temperatures(S, n, temp):
    """Masked and NaN logits have no share at any temperature; the others share alike at an infinite one."""
    rng = np.random.default_rng(n)
    x = rng.normal(0, 3, (6, n)).astype(np.float32)
    x[0, 1::2] = -np.inf
    x[1, ::3] = np.nan
    x[2] = -np.inf
    x[2, n - 1] = 0.5
    x[3, :] = np.float32(3e38)
    x[3, 1::2] = np.float32(-3e38)  # further apart than fp32's largest number
    x[4, 0], x[4, 1:] = np.float32(1e38), np.float32(-1e38)
    for kw in (dict(), dict(mp=1e-30), dict(mp=0.5)):
        with np.errstate(over="ignore"):
            want = np.stack([uncut(row, temp, kw.get("mp", 0.0)) for row in x])
        got = S.token_probs(cuda(x), cuda([temp] * 6), min_p=cuda([kw["mp"]] * 6) if kw else None).double().cpu().numpy()
        # one rounding of the share; the kept mass to n units of 2^-42 of the largest weight at worst
        assert (np.abs(got - want) <= want * (2.0 ** -24 + n * 2.0 ** -42 + 1e-12) + 2.0 ** -150).all()
        if not kw:
            # the same tokens can be drawn: the last one in the order is the last that has a share at 2
            ids, share = S.sample_rows(cuda(x), cuda([1.0 - 2.0 ** -24] * 6), cuda([temp] * 6))
            mine = torch.from_numpy(got).gather(1, ids.cpu().long()[:, None])[:, 0].numpy()
            assert (mine > 0).all() and (np.abs(mine - share.double().cpu().numpy()) <= 2.0 ** -22 * mine).all()


@pytest.mark.parametrize("n", [40, 3000, 151936])
def test_probs_min_p_below_the_bins(S, n):
    """min-p keeps tokens far below the largest with the share that they have without it, and cuts where it says."""
    rng = np.random.default_rng(n)
    x = rng.uniform(-95, 0, (8, n)).astype(np.float32)
    x[:, 0] = 0.0
    x[:, 1:30] = -np.arange(33, 91, 2, dtype=np.float32)  # weights 4.7e-15 .. 1e-38
    mp = np.array([1e-13, 1e-15, 1e-20, 1e-30, 1e-38, 1e-44, 0.0, 0.01], dtype=np.float32)
    temp = np.array([1.0, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0, 1.3], dtype=np.float32)
    for j in range(8):  # no weight within a hundred roundings of the border
        w = np.exp(x[j].astype(np.float64) / np.float64(temp[j]))
        x[j, np.abs(w - np.float64(mp[j])) <= 1e-10 * w] = -np.inf
    want = np.stack([uncut(x[j], temp[j], mp[j]) for j in range(8)])
    tol = want * (2.0 ** -24 + n * 2.0 ** -42 + 1e-12) + 2.0 ** -150
    got = S.token_probs(cuda(x), cuda(temp), min_p=cuda(mp)).double().cpu().numpy()
    assert (np.abs(got - want) <= tol).all()
    # the same through a short top-k: a top-k of the whole beginning that min-p leaves, or less
    k = np.array([min(35, n - 1)] * 8)
    order = np.argsort(-x, axis=1, kind="stable")
    for j in range(8):
        first = np.zeros(n, dtype=bool)
        first[order[j, :k[j]]] = True
        want[j] = uncut(np.where(first, x[j], -np.inf), temp[j], mp[j])
    got = S.token_probs(cuda(x), cuda(temp), top_k=cuda(k, torch.int32), min_p=cuda(mp)).double().cpu().numpy()
    assert (np.abs(got - want) <= want * (2.0 ** -24 + n * 2.0 ** -42 + 1e-12) + 2.0 ** -150).all()


def test_probs_over_the_logits_are_refused(S):
    """The logits shifted by some rows or columns, or with another stride; columns beside them are fine."""
    g = torch.Generator(device="cuda").manual_seed(2)
    rows, n = 6, 1000
    wide = torch.empty(rows + 2, 2 * n, device="cuda")
    x = wide[:rows, :n]
    x.copy_(torch.randn(rows, n, generator=g, device="cuda"))
    temp = torch.full((rows,), 0.8, device="cuda")
    want = S.token_probs(x, temp)
    for out in (x, wide[1:rows + 1, :n], wide[:rows, 1:n + 1], wide.view(-1, n)[:rows], wide[:rows, n - 1:2 * n - 1]):
        with pytest.raises(ValueError):
            S.token_probs(x, temp, out=out)
    assert torch.equal(S.token_probs(x, temp, out=wide[:rows, n:]), want)
    assert torch.equal(S.token_probs(x, temp), want)


def test_verify_starts_that_fall_are_reported(S):
    from pyrite_b200.kernels import cuda as K
    K.status()
    i32 = torch.int32
    p, x = torch.full((8, 100), 0.01, device="cuda"), cuda([3] * 8, i32)
    for starts, bad in (([0, 3, 3, 8], False), ([0, 5, 2, 8], True), ([4, 4, 8, 7], True), ([-2, 3, 3, 99], False)):
        _, counts = S.verify_drafts(p, x, cuda(starts, i32), cuda([0.0] * 8), cuda([0.5] * 3))
        torch.cuda.synchronize()
        assert K.status() == (4 if bad else 0)
        at = [min(max(s, 0), 8) for s in starts]
        assert counts.tolist() == [max(b - a, 0) for a, b in zip(at[:-1], at[1:])]  # every draft is accepted
