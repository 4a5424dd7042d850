"""Sampling on a B200 against the definition in 64 bits, row by row.

The oracle sorts a row (ties: the lower id first) and works with fp64 weights
and sums.  The kernel's weights are integers of at least 2^-42 of the largest,
so its cumulative weights differ from the oracle's by at most n * 2^-42 of the
largest weight plus fp64 noise; a row whose random number (or whose top-p
border) lies closer to a border than that may take either neighbour, and the
oracle says so.
"""
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


def oracle(row, u, temp, k, p, mp):
    """(id, probability, sharp): sharp is false within the kernel's error of a border."""
    row = np.where(np.isnan(row), -np.inf, row.astype(np.float64))
    order = np.lexsort((np.arange(row.size), -row))
    top = row[order[0]]
    if top == -np.inf:
        return -1, 0.0, True
    if not temp > 0:
        return int(order[0]), 1.0, True
    r = row[order]
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(r == top, 1.0, np.exp((r - top) / float(temp)))
    err = row.size * 2.0 ** -42 + 1e-13
    sharp = True
    n = row.size if k <= 0 else min(k, row.size)
    cum = np.cumsum(w[:n])
    if p < 1:
        target = max(float(p), 0.0) * cum[-1]
        first = int(np.searchsorted(cum, target, side="left"))
        first = min(first, n - 1)
        near = np.abs(cum - target).min()
        sharp = sharp and (near > err * 4 or target == 0.0)
        n = first + 1
    if mp > 0:
        n = min(n, int((w >= min(float(mp), 1.0)).sum()))
    cum = cum[:n]
    x = min(max(float(u), 0.0), 1.0) * cum[-1] if u > 0 else 0.0
    at = min(int(np.searchsorted(cum, x, side="right")), n - 1)
    while w[at] == 0:
        at -= 1
    sharp = sharp and (x == 0.0 or np.abs(cum - x).min() > err * 4)
    return int(order[at]), w[at] / cum[-1], sharp


def check(S, logits, u, temp, k=None, p=None, mp=None, ld=None, sharp_share=0.9):
    rows, n = logits.shape
    f = lambda x, d=torch.float32: None if x is None else torch.tensor(x, dtype=d, device="cuda")  # noqa: E731
    dev = torch.as_tensor(logits, dtype=torch.float32).cuda()
    if ld:
        wide = torch.full((rows, ld), 1e30, device="cuda")
        wide[:, :n] = dev
        dev = wide[:, :n]
    ids, probs = S.sample_rows(dev, f(u), f(temp), top_k=f(k, torch.int32), top_p=f(p), min_p=f(mp))
    ids, probs = ids.cpu().numpy(), probs.cpu().numpy()
    host = dev.cpu().numpy()
    f32 = lambda x, i, off: off if x is None else np.float32(x[i])  # noqa: E731
    sharp_rows = 0
    for j in range(rows):
        want, prob, sharp = oracle(host[j], np.float32(u[j]), np.float32(temp[j]), 0 if k is None else k[j],
                                   f32(p, j, np.float32(1)), f32(mp, j, np.float32(0)))
        if not sharp:
            continue
        sharp_rows += 1
        assert ids[j] == want, f"row {j}: {ids[j]} for {want}"
        assert abs(probs[j] - prob) <= 2.0 ** -23 * prob + n * 2.0 ** -41
    assert sharp_rows >= sharp_share * rows
    return ids


@pytest.mark.parametrize("n", [1, 2, 3, 31, 33, 128, 1000, 1025, 4097, 32000, 50257, 128256, 151936])
def test_settings_over_vocabularies(S, n):
    rng = np.random.default_rng(n)
    rows = 24
    logits = rng.normal(0, 2.5, (rows, n)).astype(np.float32)
    logits[:, rng.integers(0, n, 5)] += rng.uniform(0, 9, (rows, 5)).astype(np.float32)
    temp = rng.choice([0.0, 0.3, 0.8, 1.0, 1.7, 5.0], rows)
    k = rng.choice([0, 1, 2, 40, 1000, 5000, n, n + 7], rows).tolist()
    p = rng.choice([0.0, 0.1, 0.5, 0.9, 0.99, 0.9999, 1.0, 2.0], rows)
    mp = rng.choice([0.0, 0.0, 1e-6, 0.02, 0.3, 1.0, 1.5], rows)
    check(S, logits, rng.random(rows), temp, k, p, mp)
    check(S, logits, rng.random(rows), np.full(rows, 1.0))  # every filter off
    check(S, logits, rng.random(rows), temp, k=k)
    check(S, logits, rng.random(rows), temp, p=p)
    check(S, logits, rng.random(rows), temp, mp=mp)


@pytest.mark.parametrize("n", [7, 4096, 151936])
def test_ties(S, n):
    rng = np.random.default_rng(n + 1)
    rows = 16
    u = rng.random(rows)
    flat = np.zeros((rows, n), dtype=np.float32)  # every weight equal: the sums are exact
    flat[1::2] = -0.0
    check(S, flat, u, np.full(rows, 0.7), sharp_share=0.5)
    check(S, flat, u, np.full(rows, 1.0), k=[5] * rows, sharp_share=0.5)
    check(S, flat, u, np.full(rows, 1.0), p=np.full(rows, 0.5), sharp_share=0.0)
    coarse = np.round(rng.normal(0, 2, (rows, n)) * 2) / 2  # a few dozen distinct values
    k = [int(x) for x in rng.integers(1, n + 1, rows)]
    check(S, coarse, u, np.full(rows, 1.1), k=k)
    check(S, coarse, u, np.full(rows, 1.1), p=np.full(rows, 0.83))
    assert check(S, coarse, u, np.zeros(rows)).tolist() == [int(np.argmax(c)) for c in coarse]
    half = torch.randn(rows, n, generator=torch.Generator().manual_seed(n)).bfloat16().float().numpy()  # logits of 8 bits
    check(S, half, u, np.full(rows, 0.9), k=[50] * rows, p=np.full(rows, 0.95))
    check(S, half, u, np.full(rows, 0.9), p=np.full(rows, 0.95))


@pytest.mark.parametrize("rows,n", [(1, 300001), (2, 1 << 20), (90, 300001), (40, 50000), (80, 200)])
def test_rows_and_widths_of_every_launch(S, rows, n):
    """Few and many rows, slices that fit shared memory and slices that do not."""
    rng = np.random.default_rng(rows)
    logits = rng.normal(0, 2.0, (rows, n)).astype(np.float32)
    u = rng.random(rows)
    some = rng.choice(rows, min(rows, 12), replace=False)
    for kw in (dict(), dict(p=np.full(rows, 0.9)), dict(k=[50] * rows, p=np.full(rows, 0.9), mp=np.full(rows, 0.01)),
               dict(k=[min(n, 30000)] * rows)):
        full = {k: v for k, v in kw.items()}
        t = lambda x, d=torch.float32: torch.tensor(x, dtype=d, device="cuda")  # noqa: E731
        ids, _ = S.sample_rows(t(logits), t(u), t(np.full(rows, 0.9)), top_k=t(full["k"], torch.int32) if "k" in full else None,
                               top_p=t(full["p"]) if "p" in full else None, min_p=t(full["mp"]) if "mp" in full else None)
        ids = ids.cpu().numpy()
        sharp = 0
        for j in some:
            want, _, ok = oracle(logits[j], np.float32(u[j]), np.float32(0.9), full["k"][j] if "k" in full else 0,
                                 np.float32(full["p"][j]) if "p" in full else np.float32(1),
                                 np.float32(full["mp"][j]) if "mp" in full else np.float32(0))
            sharp += ok
            assert not ok or ids[j] == want
        assert sharp >= 0.9 * len(some)


def test_border_random_numbers(S):
    rng = np.random.default_rng(5)
    logits = rng.normal(0, 3, (8, 5000)).astype(np.float32)
    u = [0.0, -1.0, 1.0 - 2.0 ** -24, 1.0, 7.0, 2.0 ** -149, 0.5, 0.25]
    best = logits.argmax(1)
    ids = check(S, logits, u, np.ones(8), sharp_share=0.0)
    assert ids[0] == best[0] and ids[1] == best[1] and ids[5] == best[5]
    ids = check(S, logits, u, np.ones(8), k=[3] * 8, sharp_share=0.0)
    third = np.argsort(-logits, axis=1)[:, 2]
    assert ids[3] == third[3] and ids[4] == third[4]
    nan = S.sample_rows(torch.from_numpy(logits).cuda(), torch.full((8,), float("nan"), device="cuda"),
                        torch.ones(8, device="cuda"))[0]
    assert nan.cpu().tolist() == best.tolist()  # a random number that is none counts as 0


def test_masks_infinities_and_nan(S):
    n = 3001
    rng = np.random.default_rng(6)
    logits = rng.normal(0, 2, (12, n)).astype(np.float32)
    low = np.finfo(np.float32).min
    logits[0] = -np.inf                     # nothing may be taken
    logits[1] = np.nan
    logits[2, 1:] = -np.inf                 # one token
    logits[3, ::2] = -np.inf
    logits[4, 5:] = low                     # the type's lowest value as a mask
    logits[5] = low                         # ... everywhere: equal weights
    logits[6, 7] = np.inf                   # an infinite logit takes all
    logits[7, [9, 2000]] = np.inf           # two share it
    logits[8, ::3] = np.nan
    logits[9, :] = -np.inf
    logits[9, 2999] = low
    logits[10] = np.finfo(np.float32).max
    logits[10, 4:] = low
    u = rng.random(12)
    for temp in (0.0, 0.9, 1e-30, 1e30):
        for k, p, mp in ((None, None, None), ([4] * 12, np.full(12, 0.9), np.full(12, 0.01)), ([2000] * 12, None, None)):
            check(S, logits, u, np.full(12, temp), k=k, p=p, mp=mp, sharp_share=0.5)
    ids, probs = S.sample_rows(torch.from_numpy(logits).cuda(), torch.rand(12, device="cuda"),
                               torch.full((12,), float("nan"), device="cuda"))
    assert ids[0] == -1 and probs[0] == 0 and ids[1] == -1 and ids[3] % 2 == 1  # no temperature: greedy


def test_scales_and_offsets(S):
    """Logits far from zero, spread over decades, and temperatures that make one token certain or all equal."""
    rng = np.random.default_rng(7)
    base = rng.normal(0, 1, (10, 20000)).astype(np.float32)
    u = rng.random(10)
    for scale, shift in ((1e-3, 0), (30, 0), (1, 1e4), (1e6, -1e7), (1e-30, 0), (1e30, 0)):
        x = (base * np.float32(scale) + np.float32(shift)).astype(np.float32)
        for temp in (0.01, 1.0, 50.0):
            check(S, x, u, np.full(10, temp), sharp_share=0.0)
            check(S, x, u, np.full(10, temp), k=[100] * 10, p=np.full(10, 0.9), sharp_share=0.0)


def test_row_stride_stream_batch_and_capture(S):
    rng = np.random.default_rng(8)
    logits = rng.normal(0, 2.5, (200, 5003)).astype(np.float32)
    u = rng.random(200)
    check(S, logits, u, np.full(200, 0.8), k=[60] * 200, p=np.full(200, 0.97), ld=5010)
    d = torch.from_numpy(logits).cuda()
    t = torch.full((200,), 0.8, device="cuda")
    du = torch.from_numpy(u.astype(np.float32)).cuda()
    p = torch.full((200,), 0.97, device="cuda")
    base, base_p = S.sample_rows(d, du, t, top_p=p)
    for j in (0, 77, 199):  # a row's token does not depend on the batch around it
        one, one_p = S.sample_rows(d[j:j + 1], du[j:j + 1], t[:1], top_p=p[:1])
        assert int(one) == int(base[j]) and float(one_p) == float(base_p[j])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    again, _ = S.sample_rows(d, du, t, top_p=p, stream=side)
    side.synchronize()
    assert torch.equal(again, base)
    ids, probs = torch.empty_like(base), torch.empty_like(base_p)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        S.sample_rows(d, du, t, top_p=p, out=ids, probs=probs)
    du.copy_(torch.from_numpy(rng.random(200).astype(np.float32)))
    graph.replay()
    want, want_p = S.sample_rows(d, du, t, top_p=p)
    assert torch.equal(ids, want) and torch.equal(probs, want_p)


def test_frequencies(S):
    """20000 draws of one row: each token's share within five standard deviations of its probability."""
    rows = 20000
    row = torch.tensor([2.0, 1.0, 0.5, -1.0, 0.0, 3.0], device="cuda")
    u = torch.rand(rows, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    ids, _ = S.sample_rows(row.expand(rows, 6).contiguous(), u, torch.ones(rows, device="cuda"))
    p = torch.softmax(row.double(), 0).cpu()
    share = torch.bincount(ids.long(), minlength=6).double().cpu() / rows
    assert bool(((share - p).abs() <= 5 * (p * (1 - p) / rows).sqrt()).all())


@pytest.mark.parametrize("bad", ["dtype", "dim", "stride", "u", "k", "p", "out", "device"])
def test_wrapper_refuses(S, bad):
    x = torch.zeros(2, 16, device="cuda")
    v = torch.zeros(2, device="cuda")
    a = dict(logits=x, uniforms=v, temperature=v)
    a.update({"dtype": dict(logits=x.half()), "dim": dict(logits=x[0]), "stride": dict(logits=x[:, ::2]),
              "u": dict(uniforms=v[:1]), "k": dict(top_k=v), "p": dict(top_p=v.double()),
              "out": dict(out=torch.zeros(2, device="cuda")), "device": dict(temperature=v.cpu())}[bad])
    with pytest.raises(ValueError):
        S.sample_rows(**a)


@pytest.mark.parametrize("n", [7, 4096, 50000, 151936, 300001, 1 << 20])
@pytest.mark.parametrize("rows", [3, 80])
def test_equal_weights_are_exact(S, n, rows):
    """Equal logits: every weight is 2^S units, so kept tokens and the pick are whole numbers, at every width.
    top_p keeps the tokens j with j < top_p * n, the pick is the first j with j + 1 > u * kept."""
    from fractions import Fraction
    rows = min(rows, max(3, (80 << 18) // n))
    rng = np.random.default_rng(n)
    logits = torch.full((rows, n), -3.5, device="cuda")
    u = rng.random(rows).astype(np.float32)
    temp = torch.full((rows,), 0.7, device="cuda")
    for p in (0.5, 0.25, 1.0, float(np.float32(0.3))):
        ids, probs = S.sample_rows(logits, torch.from_numpy(u).cuda(), temp,
                                   top_p=torch.full((rows,), p, device="cuda"))
        kept = min(n, -(-(Fraction(p) * n) // 1))
        want = [int(Fraction(float(x)) * kept) for x in u]
        # u has 24 bits and kept at most 20, so u * kept * 2^S is exact in 53 bits; the share is rounded twice
        assert ids.tolist() == want
        assert bool(((probs.double().cpu() * int(kept) - 1).abs() <= 2.0 ** -23).all())


def test_differences_past_the_largest_float(S):
    """A token whose logit lies more than fp32's largest number below the row's largest counts as -inf, whatever the
    temperature; nearer ones weigh by the formula."""
    n = 4000
    rng = np.random.default_rng(9)
    logits = rng.choice(np.float32([3.2e38, 2.9e38, 1.0e38, 1.5e37, 0.0]), (16, n)).astype(np.float32)
    far = logits.copy()
    far[:, rng.choice(n, n // 2, replace=False)] = np.float32(-3.0e38)
    u = rng.random(16).astype(np.float32)
    ones = torch.ones(16, device="cuda")
    for temp in (1e36, 1e37, 1e38, 3e38, float("inf")):
        for kw in (dict(), dict(p=np.full(16, 0.8)), dict(k=[600] * 16)):
            full = check(S, logits, u, np.full(16, temp), **kw)
            assert full.min() >= 0
            masked = np.where(far < -1e38, np.float32(-np.inf), far)
            args = dict(top_p=None if "p" not in kw else ones * 0.8,
                        top_k=None if "k" not in kw else torch.full((16,), 600, dtype=torch.int32, device="cuda"))
            got = [S.sample_rows(torch.from_numpy(x).cuda(), torch.from_numpy(u).cuda(), ones * temp, **args)
                   for x in (far, masked)]
            assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
