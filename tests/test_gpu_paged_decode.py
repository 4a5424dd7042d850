"""Serving requests of different lengths behind a shared prefix (PagedDecoder, B200).

The oracle of greedy requests is one single-sequence decode of prefix + prompt
per request (MixedDecoder.generate, itself checked against the reference
executor's ids); sampled requests are compared with the 64-bit definition on
the decoder's own logits, step by step.
"""
from __future__ import annotations

import json
from dataclasses import fields
from pathlib import Path

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

GOLDEN = Path(__file__).resolve().parent / "golden"


def make(golden, device, **kw):
    from pyrite_b200.paged import PagedDecoder
    from pyrite_b200.synthetic import DenseSpec, MoESpec
    g = json.loads((GOLDEN / golden).read_text())
    cls = MoESpec if g["spec"]["architecture"] == "qwen3moe" else DenseSpec
    spec = cls(**{k: v for k, v in g["spec"].items() if k in {f.name for f in fields(cls)}})
    return g, spec, PagedDecoder.synthetic(spec, device=device, **kw)


def prompts_of(spec, lengths, seed):
    rng = np.random.default_rng(seed)
    return [[int(t) for t in rng.integers(0, spec.vocab_size, n)] for n in lengths]


@pytest.mark.parametrize("golden", ["llama_tiny.json", "moe_tiny.json"])
def test_ragged_greedy_requests_equal_single_runs(cuda_device, golden):
    g, spec, dec = make(golden, cuda_device, max_ctx=96, batch=5)
    prompts = [g["prompt"]] + prompts_of(spec, [1, 17, 5, 30], 1)
    new = [len(g["generated"]), 9, 4, 20, 1]
    got = dec.pgenerate(prompts, new)
    assert got[0][len(g["prompt"]):] == g["generated"], "request 0 differs from the reference executor"
    for p, m, have in zip(prompts, new, got):
        assert have == dec.generate(p, m)
    # again with fewer requests, other settings of the same decoder and prompts in blocks
    got = dec.pgenerate(prompts[1:4], 6, prefill_block=8)
    for p, have in zip(prompts[1:4], got):
        assert have == dec.generate(p, 6)
    assert dec.bgenerate(prompts[:2], 3) == [dec.generate(p, 3) for p in prompts[:2]]


@pytest.mark.parametrize("golden", ["llama_tiny.json", "moe_tiny.json"])
@pytest.mark.parametrize("prefix_len", [1, 16, 37])
def test_requests_behind_a_shared_prefix(cuda_device, golden, prefix_len):
    g, spec, dec = make(golden, cuda_device, max_ctx=96, batch=4)
    prefix = prompts_of(spec, [prefix_len], 2)[0]
    prompts = prompts_of(spec, [3, 18, 1, 11], 3)
    dec.set_prefix(prefix)
    for block in (0, 7):
        got = dec.pgenerate(prompts, 8, prefill_block=block)
        for p, have in zip(prompts, got):
            want = dec.generate(prefix + p, 8)  # this overwrites the one-sequence caches; the pages keep the prefix
            assert have == want[prefix_len:]
    dec.set_prefix([])
    assert dec.pgenerate(prompts[:1], 5) == [dec.generate(prompts[0], 5)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_16_bit_caches(cuda_device, dtype):
    """The logits of a 16-bit cache stay near the fp32 cache's: keys and values rounded to half a step."""
    g, spec, exact = make("llama_tiny.json", cuda_device, max_ctx=64, batch=3)
    _, _, dec = make("llama_tiny.json", cuda_device, max_ctx=64, batch=3, kv_dtype=dtype, page_size=32)
    prompts = prompts_of(spec, [20, 9, 33], 4)
    prefix = prompts_of(spec, [13], 5)[0]
    out = []
    for d in (exact, dec):
        d.set_prefix(prefix)
        d.pgenerate(prompts, 1)
        out.append(d.blogits[2].clone())  # the longest request's last step
    step = torch.finfo(dtype).eps / 2
    # relative to the logits' size: some layers' worth of half steps
    assert float((out[1] - out[0]).norm() / out[0].norm()) <= 8 * step * spec.num_hidden_layers


def test_sampled_requests_follow_the_definition(cuda_device):
    from tests.test_gpu_sampling import oracle
    g, spec, dec = make("llama_tiny.json", cuda_device, max_ctx=64, batch=4)
    prompts = prompts_of(spec, [2, 6, 6, 3], 6)
    u = torch.rand(4, 64, generator=torch.Generator().manual_seed(1))
    sets = dict(temperature=[0.8, 1.0, 0.0, 1.5], top_k=[0, 20, 0, 5], top_p=[0.9, 1.0, 1.0, 0.99],
                min_p=[0.0, 0.02, 0.0, 0.0])
    # one token at a time: a run of m tokens ends on the logits that gave token m
    for m in (1, 2, 5):
        got = dec.pgenerate([p for p in prompts], m, uniforms=u, **sets)
        logits = dec.blogits.cpu().numpy()
        for j in (1, 2):  # the longest prompts take the run's last step
            t = len(prompts[j]) + m - 1
            want, _, sharp = oracle(logits[j], np.float32(u[j, t]), np.float32(sets["temperature"][j]),
                                    sets["top_k"][j], np.float32(sets["top_p"][j]), np.float32(sets["min_p"][j]))
            assert not sharp or got[j][-1] == want
    a, b = dec.pgenerate(prompts, 12, temperature=1.0, seed=5), dec.pgenerate(prompts, 12, temperature=1.0, seed=5)
    assert a == b and a != dec.pgenerate(prompts, 12, temperature=1.0, seed=6)
    # the same draws whether the prompt ran step by step or in blocks
    assert dec.pgenerate(prompts, 4, uniforms=u, **sets) == dec.pgenerate(prompts, 4, uniforms=u, prefill_block=4, **sets)


def test_pages_are_handed_out_as_requests_grow(cuda_device):
    g, spec, dec = make("llama_tiny.json", cuda_device, max_ctx=64, batch=3, n_pages=6)
    prompts = prompts_of(spec, [15, 1, 20], 7)
    dec.pgenerate(prompts, [2, 1, 13])  # 16, 1 and 32 cached tokens: one, one and two pages
    assert dec.lens.tolist() == [16, 1, 32] and int(dec.used) == 4
    assert (dec.table >= 0).sum(1).tolist() == [1, 1, 2]
    with pytest.raises(ValueError, match="pages"):
        dec.pgenerate(prompts_of(spec, [40, 40, 20], 8), 5)


@pytest.mark.parametrize("call", [
    lambda d: d.pgenerate([], 3), lambda d: d.pgenerate([[1]] * 4, 3), lambda d: d.pgenerate([[]], 3),
    lambda d: d.pgenerate([[1, 10 ** 7]], 3), lambda d: d.pgenerate([[1] * 30], 3), lambda d: d.pgenerate([[1]], 0),
    lambda d: d.pgenerate([[1], [2]], [3]), lambda d: d.pgenerate([[1], [2]], 3, temperature=[1.0]),
    lambda d: d.pgenerate([[1]], 3, uniforms=torch.rand(1, 2)), lambda d: d.set_prefix([-1]),
    lambda d: d.set_prefix([1] * 31)])
def test_refusals(cuda_device, call):
    if not hasattr(test_refusals, "dec"):
        test_refusals.dec = make("llama_tiny.json", cuda_device, max_ctx=32, batch=3)[2]
    with pytest.raises(ValueError):
        call(test_refusals.dec)


def test_a_request_without_a_token_to_take_is_reported(cuda_device):
    """Logits that are all NaN give no token (-1): an error, never made-up tokens."""
    g, spec, dec = make("llama_tiny.json", cuda_device, max_ctx=48, batch=3)
    prompts = prompts_of(spec, [4, 1, 9], 11)
    want = dec.pgenerate(prompts, [5, 2, 3])
    norm = dec.out_norm.clone()
    dec.out_norm.fill_(float("nan"))
    for sampled in (dict(), dict(temperature=1.0, top_p=0.9)):
        with pytest.raises(RuntimeError, match=r"\[0, 1, 2\]"):
            dec.pgenerate(prompts, [5, 2, 3], **sampled)
    dec.out_norm.copy_(norm)
    assert dec.pgenerate(prompts, [5, 2, 3]) == want


@pytest.mark.parametrize("fails", ["store_kv", "page_tables"])
def test_a_prefix_that_fails_leaves_no_prefix(cuda_device, monkeypatch, fails):
    """A set_prefix that raises leaves a decoder without prefix, also where the old one had the same length."""
    from pyrite_b200.kernels import paged
    g, spec, dec = make("llama_tiny.json", cuda_device, max_ctx=64, batch=2)
    old, new = prompts_of(spec, [20, 20], 12)
    prompts = prompts_of(spec, [3, 7], 13)
    dec.set_prefix(old)
    dec.pgenerate(prompts, 6)

    def refuse(*a, **kw):
        raise RuntimeError("no memory")

    with monkeypatch.context() as m:
        m.setattr(paged, fails, refuse)
        with pytest.raises(RuntimeError, match="no memory"):
            dec.set_prefix(new)
    assert dec.pgenerate(prompts, 6) == [dec.generate(p, 6) for p in prompts]
    dec.set_prefix(new)
    assert dec.pgenerate(prompts, 6) == [dec.generate(new + p, 6)[20:] for p in prompts]


@pytest.mark.parametrize("golden", ["llama_tiny.json", "moe_tiny.json"])
def test_ended_requests_attend_to_nothing(cuda_device, golden):
    """A request that has ended, and a row without one, reads no key of its own in the steps of the others."""
    g, spec, dec = make(golden, cuda_device, max_ctx=96, batch=4)
    prompts = prompts_of(spec, [30, 2, 17], 14)
    got = dec.pgenerate(prompts, [3, 50, 1])
    assert dec.fresh.tolist() == [0, 0, 0, 0] and dec.lens.tolist() == [32, 51, 17, 0]
    assert not bool(dec.batt[[0, 2, 3]].any()) and bool(dec.batt[1].any())  # of the last step, its last layer
    for p, m, have in zip(prompts, [3, 50, 1], got):
        assert have == dec.generate(p, m)
