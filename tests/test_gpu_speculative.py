"""The operators of a serving loop one after the other, on a small model of one attention layer: prompts in
chunks behind a shared prefix, requests forked from them, drafted tokens appended, attended to, verified and
the refused ones given back -- against one-token-at-a-time greedy decoding in fp64.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

HD, NQ, NKV, HID, VOCAB, PS = 128, 8, 2, 64, 300, 16


@pytest.fixture(scope="module")
def K(cuda_device):
    from pyrite_b200.kernels import cuda
    cuda.status()
    return cuda


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def rope_table(n):
    inv = 1e4 ** (-2.0 * np.arange(64) / HD)
    ang = np.arange(n)[:, None] * inv[None, :]
    return torch.from_numpy(np.ascontiguousarray(np.stack([np.cos(ang), np.sin(ang)], -1))).cuda()


class Model:
    """logits of a token = W_out attention(q, k, v of the tokens so far); all of a token's q, k, v from its embedding."""

    def __init__(self, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.embed = torch.randn(VOCAB, HID, generator=g, device="cuda")
        self.w_qkv = torch.randn(HID, (NQ + 2 * NKV) * HD, generator=g, device="cuda") / math.sqrt(HID) * 1.3
        self.w_out = torch.randn(NQ * HD, VOCAB, generator=g, device="cuda") / 8
        self.rope = rope_table(512)

    def qkv(self, tokens):
        return self.embed[tokens.long()] @ self.w_qkv

    def greedy(self, tokens, n, dtype):
        """fp64, keys and values rounded to the cache's type: n greedy tokens and the smallest gap to the second."""
        out, gap = list(tokens), float("inf")
        for _ in range(n):
            x = self.qkv(torch.tensor(out, device="cuda")).double().view(len(out), NQ + 2 * NKV, HD)
            cs = self.rope[:len(out)][:, None]

            def rot(y):
                a, b = y[..., :64], y[..., 64:]
                return torch.cat([a * cs[..., 0] - b * cs[..., 1], a * cs[..., 1] + b * cs[..., 0]], -1)

            q, k = rot(x[:, :NQ])[-1], rot(x[:, NQ:NQ + NKV]).to(dtype).double()
            v = x[:, NQ + NKV:].to(dtype).double()
            s = torch.einsum("hgd,thd->hgt", q.view(NKV, NQ // NKV, HD), k) / math.sqrt(HD)
            o = torch.einsum("hgt,thd->hgd", torch.softmax(s, -1), v).reshape(-1)
            two, ids = torch.topk(o @ self.w_out.double(), 2)
            gap = min(gap, float(two[0] - two[1]))
            out.append(int(ids[0]))
        return out[len(tokens):], gap


@pytest.mark.parametrize("dtype,guess_right", [(torch.float32, 0.7), (torch.float16, 0.6), (torch.bfloat16, 0.0),
                                               (torch.float16, 1.0)])
def test_drafts_verified_over_a_forked_paged_cache(K, dtype, guess_right):
    from pyrite_b200.kernels import paged, sampling
    model, rng = Model(1), np.random.default_rng(2)
    prefix = rng.integers(0, VOCAB, 21).tolist()
    prompts = [rng.integers(0, VOCAB, n).tolist() for n in (37, 16, 5)]
    parents, want_new, drafts = [-1, -1, -1, 0, 0, 1, 2], 24, 4
    R = len(parents)
    n_pages = 80
    pool = paged.KVPool.zeros(n_pages, NKV, PS, dtype)
    free, used = ints(rng.permutation(n_pages)), ints([0])
    table, shared = torch.full((R, 12), -1, dtype=torch.int32, device="cuda"), torch.zeros(n_pages, dtype=torch.int32, device="cuda")
    pre_table = torch.full((1, 4), -1, dtype=torch.int32, device="cuda")
    lens = ints([0] * R)

    def chunk(tokens, counts, first, tbl, lens_now, prefix_len):
        """Rows of `tokens`, counts[i] of request i, appended and attended to; their logits and the new lengths."""
        n = int(sum(counts))
        slots = paged.TokenSlots.empty(len(counts), capacity=n)
        paged.page_tables(lens_now, ints(counts), PS, free, used, tbl, slots)
        q = paged.append_kv(model.qkv(tokens), pool, slots.slots, slots.positions, model.rope, NQ, first=first)
        o = paged.attention_chunks(q, pool, tbl, slots.starts, slots.kv_lens, prefix_pages=pre_table[0],
                                   prefix_len=prefix_len)
        return o @ model.w_out, slots

    # the prefix, once
    chunk(ints(prefix), [len(prefix)], 0, pre_table, ints([0]), 0)
    held = int(used)
    assert held == 2
    # the prompts in two chunks each, all but their last tokens
    for part in (0, 1):
        cut = [p[:len(p) // 2] if part == 0 else p[len(p) // 2:-1] for p in prompts]
        counts = [len(c) for c in cut] + [0] * (R - 3)
        if sum(counts):
            _, slots = chunk(ints(sum(cut, [])), counts, len(prefix), table, lens, len(prefix))
            lens = slots.kv_lens.clone()
    # samples of one prompt continue it
    copies = paged.fork_requests(ints(parents), lens, PS, free, used, table, shared)
    paged.copy_pages([pool], copies)
    of = [i if p < 0 else p for i, p in enumerate(parents)]
    assert lens.tolist() == [len(prompts[p]) - 1 for p in of]
    want, gap = [], float("inf")
    for p in prompts:
        w, g = model.greedy(prefix + p, want_new + drafts, dtype)
        want.append(w)
        gap = min(gap, g)
    assert gap > 1e-3  # far above what the kernels' roundings move a logit (1e-5 of logits of some units)
    current, got = [prompts[p][-1] for p in of], [[] for _ in range(R)]
    greedy = torch.zeros(1, device="cuda")
    steps = 0
    while min(len(g) for g in got) < want_new:
        live = [i for i in range(R) if len(got[i]) < want_new]
        counts = [0] * R
        rows, ahead = [], []
        for i in live:
            k = int(rng.integers(0, drafts + 1))  # some requests draft nothing
            guess = [t if rng.random() < guess_right else int(rng.integers(0, VOCAB))
                     for t in want[of[i]][len(got[i]):len(got[i]) + k]]
            rows += [current[i]] + guess
            ahead += guess + [-1]
            counts[i] = k + 1
        logits, slots = chunk(ints(rows), counts, len(prefix), table, lens, len(prefix))
        probs = sampling.token_probs(logits, greedy.expand(len(rows)).contiguous())
        tokens, n = sampling.verify_drafts(probs, ints(ahead), slots.starts, torch.rand(len(rows), device="cuda"),
                                           torch.rand(R, device="cuda"))
        # tokens kept: the one that was run and the accepted drafts; the last new one is run next
        keep = lens + n
        paged.release_pages(slots.kv_lens, keep, PS, free, used, table, shared)
        lens = slots.kv_lens
        starts, tokens, n = slots.starts.tolist(), tokens.tolist(), n.tolist()
        for i in live:
            new = tokens[starts[i]:starts[i] + n[i]]
            assert n[i] >= 1 and -1 not in new
            got[i] += new
            current[i] = new[-1]
        steps += 1
    torch.cuda.synchronize()
    assert K.status() == 0
    for i in range(R):
        assert got[i][:want_new] == want[of[i]][:want_new], i
    if guess_right == 1.0:
        assert steps < want_new  # accepted drafts save steps
    # every page comes back
    paged.release_pages(lens, ints([0] * R), PS, free, used, table, shared)
    torch.cuda.synchronize()
    assert int(used) == held and not bool(shared.any()) and K.status() == 0
    assert sorted(free.tolist()) == list(range(n_pages))


def test_settings_of_requests_for_rows_that_vary(K):
    """Temperatures and filters of each request, looked up for its rows on the device: one graph for all splits."""
    from pyrite_b200.kernels import sampling
    g = torch.Generator(device="cuda").manual_seed(3)
    R, rows, n = 6, 20, 3000
    temperature, top_k = torch.tensor([0.0, 0.7, 1.3, 0.0, 0.9, 2.0], device="cuda"), ints([0, 40, 0, 5, 700, 3])
    top_p, logits = torch.tensor([1.0, 0.9, 0.5, 1.0, 0.8, 1.0], device="cuda"), torch.randn(rows, n, device="cuda", generator=g) * 3
    drafts, accept = torch.randint(0, n, (rows,), generator=g, device="cuda").int(), torch.rand(rows, device="cuda", generator=g)
    pick, starts, number = torch.rand(R, device="cuda", generator=g), ints([0] * (R + 1)), torch.arange(rows, device="cuda")

    def step():
        row_of = torch.searchsorted(starts[1:], number, right=True).clamp(max=R - 1)
        p = sampling.token_probs(logits, temperature[row_of], top_k=top_k[row_of], top_p=top_p[row_of])
        return p, *sampling.verify_drafts(p, drafts, starts, accept, pick)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for counts in ([4, 3, 5, 1, 2, 5], [0, 0, 9, 0, 8, 3], [20, 0, 0, 0, 0, 0], [1, 2, 0, 4, 0, 0]):
        host = np.concatenate([[0], np.cumsum(counts)])
        starts.copy_(ints(host.tolist()))
        graph.replay()
        of = np.repeat(np.arange(R), counts).tolist()
        m = len(of)
        want = sampling.token_probs(logits[:m], temperature[of], top_k=top_k[of], top_p=top_p[of])
        tokens, n_tokens = sampling.verify_drafts(want, drafts[:m], starts, accept[:m], pick)
        torch.cuda.synchronize()
        assert K.status() == 0
        assert torch.equal(out[0][:m], want) and torch.equal(out[1][:m], tokens) and torch.equal(out[2], n_tokens)
